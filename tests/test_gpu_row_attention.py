"""Tree attention and weight attention on the device against their 64-bit forms (row_reference.py derives the bounds)."""

from __future__ import annotations

import math

import pytest
import torch

from logkv_amd import log_kv_tree_attention, log_kv_weight_attention
from row_reference import check_close, reference, tree_mask

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def rows(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def inputs(B, G, rep, T, cap, dk, dv, dtype, seed, layout="rows"):
    q, k, v = rows((B, G * rep, T, dk), dtype, seed, 2.0), rows((B, G, T, dk), dtype, seed + 1), rows((B, G, T, dv), dtype, seed + 2)
    if layout == "rows":
        ck, cv = rows((B, G, cap, dk), dtype, seed + 3), rows((B, G, cap, dv), dtype, seed + 4)
    elif layout == "padded":      # features of wider rows
        ck, cv = (rows((B, G, cap, d + 8), dtype, seed + 3 + i)[..., :d] for i, d in enumerate((dk, dv)))
        q = rows((B, T, G * rep, dk + 8), dtype, seed, 2.0)[..., :dk].transpose(1, 2)
        k, v = (rows((B, T, G, d + 16), dtype, seed + 1 + i)[..., 8:8 + d].transpose(1, 2) for i, d in enumerate((dk, dv)))
    else:                         # tokens before heads; odd strides that the call has to copy for its own rows
        ck, cv = (rows((B, cap, G, d), dtype, seed + 3 + i).transpose(1, 2) for i, d in enumerate((dk, dv)))
        q = rows((B, G * rep, T, dk + 1), dtype, seed, 2.0)[..., 1:]
    return q, k, v, ck, cv


TREES = [
    # B, G, rep, T, lengths, cap, dk, dv, dtype, layout
    (1, 1, 1, 1, [1], 1, 64, 64, BF16, "rows"),
    (1, 2, 2, 1, [0], 8, 64, 64, BF16, "rows"),
    (2, 2, 2, 8, [33, 31], 40, 128, 128, BF16, "rows"),
    (2, 2, 2, 8, [32, 64], 64, 128, 128, F16, "padded"),
    (1, 2, 3, 13, [129], 130, 80, 80, BF16, "tokens"),
    (3, 1, 1, 33, [500, 1, 0], 512, 96, 96, F16, "rows"),
    (1, 2, 2, 26, [900], 901, 128, 128, BF16, "padded"),
    (2, 1, 8, 9, [257, 300], 300, 64, 64, F16, "tokens"),
    (1, 2, 8, 40, [333], 333, 128, 64, BF16, "rows"),
    (1, 1, 5, 61, [640], 700, 64, 64, F16, "rows"),
    (1, 1, 2, 7, [70], 70, 192, 128, BF16, "rows"),
    (2, 1, 2, 20, [100, 37], 128, 256, 256, BF16, "padded"),
    (1, 1, 3, 50, [150], 160, 256, 200, F16, "rows"),
    (1, 1, 1, 3, [10], 12, 8, 8, BF16, "rows"),
    (1, 2, 4, 100, [1100], 1100, 128, 128, BF16, "rows"),
    (1, 1, 2, 150, [2000], 2048, 128, 128, F16, "rows"),
]


@pytest.mark.parametrize("B,G,rep,T,lengths,cap,dk,dv,dtype,layout", TREES)
def test_tree_attention(B, G, rep, T, lengths, cap, dk, dv, dtype, layout):
    q, k, v, ck, cv = inputs(B, G, rep, T, cap, dk, dv, dtype, 7 * T + cap, layout)
    visible = torch.stack([tree_mask(T, 11 + b, empty=(T - 1,) if T > 2 else ()) for b in range(B)])
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    scale = dk ** -0.5
    before = ck.clone(), cv.clone()
    out = log_kv_tree_attention(q, k, v, ck, cv, n, visible.cuda(), scale)
    want, _, bound, _ = reference(q, k, v, ck, cv, lengths, visible, scale)
    check_close(out, want, bound)
    assert torch.equal(ck, before[0]) and torch.equal(cv, before[1])
    # One mask for the whole batch, as bytes, and the length as a number.
    if len(set(lengths)) == 1:
        shared = log_kv_tree_attention(q, k, v, ck, cv, lengths[0], visible[0].to(torch.uint8).cuda(), scale)
        want, _, bound, _ = reference(q, k, v, ck, cv, lengths, visible[:1].expand(B, T, T), scale)
        check_close(shared, want, bound)


@pytest.mark.parametrize("kind", ["float", "half", "packed"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rep,T", [(2, 3), (2, 20), (4, 40)])
def test_tree_bias(kind, dtype, rep, T):
    B, G, cap, d = 2, 2, 210, 64
    lengths = [200, 77]
    q, k, v, ck, cv = inputs(B, G, rep, T, cap, d, d, dtype, 5)
    log_mass = torch.log(torch.floor(torch.rand(B, G, cap, generator=torch.Generator().manual_seed(3)) * 63 + 1))
    lowest = torch.finfo(torch.float32 if kind == "float" else dtype).min
    log_mass[:, :, 5::17] = -math.inf
    log_mass[:, :, 7::19] = lowest
    if kind == "float":
        bias = log_mass.cuda()
    elif kind == "half":
        bias = log_mass.to(dtype).cuda().transpose(1, 2).contiguous().transpose(1, 2)
    else:
        packed = torch.zeros(B, G, cap, d + 8, dtype=dtype, device="cuda")
        packed[..., :d], packed[..., d] = ck, log_mass.to(dtype).cuda()
        ck, bias = packed[..., :d], packed[..., d]
    # What hidden rows hold reaches nothing: rows hidden by the bias, rows behind the last.
    ck[:, :, 5::17], cv[:, :, 5::17] = math.nan, math.inf
    for b, n in enumerate(lengths):
        ck[b, :, n:], cv[b, :, n:], bias[b, :, n:] = math.nan, math.nan, math.nan
    visible = tree_mask(T, 4)[None].expand(B, T, T)
    out = log_kv_tree_attention(q, k, v, ck, cv, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                visible[0].cuda(), d ** -0.5, bias=bias)
    want, _, bound, _ = reference(q, k, v, ck, cv, lengths, visible, d ** -0.5, bias)
    assert bool(torch.isfinite(want).all())
    check_close(out, want, bound)


def test_tree_all_rows_hidden():
    """Only hidden rows in the cache (-inf) and no visible drafted row: zeros; the lowest value hides nothing by itself."""
    q, k, v, ck, cv = inputs(1, 1, 2, 4, 40, 64, 64, BF16, 9)
    visible = torch.zeros(4, 4, dtype=torch.bool)
    visible[2, 0] = True
    hidden = torch.full((1, 1, 40), -math.inf, device="cuda")
    out = log_kv_tree_attention(q, k, v, ck, cv, 40, visible.cuda(), 0.125, bias=hidden)
    want, _, bound, _ = reference(q, k, v, ck, cv, [40], visible[None], 0.125, hidden)
    check_close(out, want, bound)
    assert bool((out[:, :, [0, 1, 3]] == 0).all()) and bool((out[:, :, 2] == v[:, :, 0]).all())
    lowest = torch.full((1, 1, 40), torch.finfo(torch.float32).min, device="cuda")
    out = log_kv_tree_attention(q, k, v, ck, cv, 40, torch.zeros_like(visible).cuda(), 0.125, bias=lowest)
    assert bool(torch.isfinite(out.float()).all()) and bool((out != 0).any())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rep,T,d", [(2, 5, 64), (2, 12, 128), (4, 40, 128), (2, 9, 256)])
def test_infinities_reach_only_who_sees_them(dtype, rep, T, d):
    G, cap = 2, 70
    q, k, v, ck, cv = inputs(1, G, rep, T, cap, d, d, dtype, 21)
    visible = tree_mask(T, 2)
    v[0, 0, 1, 3], v[0, 0, 2, 4], v[0, 1, 0, 5] = math.inf, -math.inf, math.nan
    k[0, 1, T - 1, 0] = math.nan
    out = log_kv_tree_attention(q, k, v, ck, cv, 65, visible.cuda(), d ** -0.5)
    want, _, bound, _ = reference(q, k, v, ck, cv, [65], visible[None], d ** -0.5)
    assert bool(torch.isinf(want).any()) and bool(torch.isnan(want).any()) and bool(torch.isfinite(want[0, 0, 0]).all())
    check_close(out, want, bound)
    # In a row of the cache: everyone sees it.
    q, k, v, ck, cv = inputs(1, G, rep, T, cap, d, d, dtype, 22)
    cv[0, 0, 40, 2], cv[0, 0, 41, 2], cv[0, 0, 3, 1] = math.inf, -math.inf, -math.inf
    out = log_kv_tree_attention(q, k, v, ck, cv, 65, visible.cuda(), d ** -0.5)
    want, _, bound, _ = reference(q, k, v, ck, cv, [65], visible[None], d ** -0.5)
    check_close(out, want, bound)


@pytest.mark.parametrize("dtype,size", [(BF16, 1e-30), (BF16, 1e-9), (BF16, 1e-3), (BF16, 700.0), (BF16, 1e25), (BF16, "mixed"),
                                        (F16, 1e-6), (F16, 1e-3), (F16, 2e4), (F16, "mixed")])
@pytest.mark.parametrize("rep,T", [(2, 4), (2, 20), (2, 40), (4, 50)])
def test_value_magnitudes(dtype, size, rep, T):
    """Values of any exponent: tiny, huge (fp16: some beyond its range, infinite), and features of very different sizes in one row (some tiles with a huge row)."""
    d, cap = 64, 300
    q, k, v, ck, cv = inputs(1, 1, rep, T, cap, d, d, torch.float32, 25)
    if size == "mixed":
        power = torch.arange(d, device="cuda") % 16 * (2.0 if dtype == BF16 else 0.8) - 24.0 * (dtype == BF16) - 8.0 * (dtype == F16)
        v, cv = v * 2.0 ** power, cv * 2.0 ** power
        cv[:, :, 200] *= 2.0 ** (14 if dtype == BF16 else 10)
    else:
        v, cv = v * size, cv * size
    q, k, v, ck, cv = (x.to(dtype) for x in (q, k, v, ck, cv))
    visible = tree_mask(T, 6)
    out = log_kv_tree_attention(q, k, v, ck, cv, cap, visible.cuda(), d ** -0.5)
    want, _, bound, _ = reference(q, k, v, ck, cv, [cap], visible[None], d ** -0.5)
    check_close(out, want, bound + 1e-38)


WEIGHTS = [
    (1, 1, 1, 1, [1], 2, 64, 64, BF16, "rows"),
    (1, 2, 2, 1, [0], 8, 64, 64, BF16, "rows"),
    (2, 2, 2, 1, [33, 31], 40, 128, 128, BF16, "rows"),
    (2, 2, 4, 2, [1000, 517], 1100, 96, 96, F16, "padded"),
    (1, 2, 8, 2, [2049], 2060, 128, 128, BF16, "rows"),
    (1, 2, 16, 1, [300], 301, 128, 64, F16, "rows"),
    (2, 1, 3, 5, [100, 64], 128, 80, 80, BF16, "tokens"),
    (1, 1, 2, 33, [100], 140, 64, 64, BF16, "padded"),
    (1, 1, 4, 70, [500], 570, 128, 128, F16, "rows"),
    (2, 1, 2, 333, [700, 0], 1100, 64, 64, BF16, "rows"),
    (1, 1, 2, 9, [70], 79, 192, 128, BF16, "rows"),
    (1, 1, 2, 40, [70], 120, 256, 256, F16, "rows"),
    (1, 1, 1, 300, [1300], 1600, 128, 128, BF16, "rows"),
]


@pytest.mark.parametrize("B,G,rep,T,lengths,cap,dk,dv,dtype,layout", WEIGHTS)
def test_weight_attention(B, G, rep, T, lengths, cap, dk, dv, dtype, layout):
    q, k, v, ck, cv = inputs(B, G, rep, T, cap, dk, dv, dtype, 3 * T + cap, layout)
    w = torch.rand(B, G, cap, generator=torch.Generator().manual_seed(8)).cuda()
    w0, k0, v0 = w.clone(), ck.clone(), cv.clone()
    scale = dk ** -0.5
    causal = torch.ones(T, T, dtype=torch.bool).tril()[None].expand(B, T, T)
    want, column, bound, rel = reference(q, k, v, ck, cv, lengths, causal, scale)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = log_kv_weight_attention(q, k, v, ck, cv, w, n, scale)
    check_close(out, want, bound)
    for b, m in enumerate(lengths):
        stored = min(T, cap - m)
        total = w0[b].cpu().double()
        total[:, :m] += column[b, :, :m]
        total[:, m:m + stored] = column[b, :, cap:cap + stored]
        # Sums of rep T probabilities and the weight before, in float32.
        check_close(w[b], total, (rel + (rep * T + 2) * 2.0 ** -24) * column[b][:, list(range(m)) + list(range(cap, cap + stored))
                    + [0] * (cap - m - stored)].abs() + 2.0 ** -23 * total.abs() + 1e-30, f"weights of row {b}")
        assert torch.equal(w[b, :, m + stored:], w0[b, :, m + stored:])
        for cache, old, new in ((ck, k0, k), (cv, v0, v)):
            assert torch.equal(cache[b, :, :m], old[b, :, :m]) and torch.equal(cache[b, :, m + stored:], old[b, :, m + stored:])
            assert torch.equal(cache[b, :, m:m + stored], new[b, :, :stored])
    # The same call on the same state gives the same bits.
    w2, ck2, cv2 = w0.clone(), k0, v0
    out2 = log_kv_weight_attention(q, k, v, ck2, cv2, w2, n, scale)
    assert torch.equal(out, out2) and torch.equal(w, w2) and torch.equal(ck, ck2) and torch.equal(cv, cv2)


@pytest.mark.parametrize("T,rep", [(4, 2), (50, 2)])
def test_weight_counts_of_a_padded_batch(T, rep):
    B, G, cap, d = 4, 2, 200, 64
    lengths, counts = [10, 0, 100, 64], [T, 1, 0, T - 1]
    q, k, v, ck, cv = inputs(B, G, rep, T, cap, d, d, BF16, 31)
    for b, c in enumerate(counts):   # padding holds anything
        q[b, :, c:], k[b, :, c:], v[b, :, c:] = math.nan, math.nan, math.inf
    w = torch.rand(B, G, cap, device="cuda")
    w0, k0 = w.clone(), ck.clone()
    causal = torch.ones(T, T, dtype=torch.bool).tril()[None].expand(B, T, T)
    want, column, bound, rel = reference(q, k, v, ck, cv, lengths, causal, 0.125, counts=counts)
    out = log_kv_weight_attention(q, k, v, ck, cv, w, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0.125,
                                  counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
    check_close(out, want, bound)
    for b, (m, c) in enumerate(zip(lengths, counts)):
        assert bool((out[b, :, c:] == 0).all())
        total = w0[b].cpu().double()
        total[:, :m] += column[b, :, :m]
        total[:, m:m + c] = column[b, :, cap:cap + c]
        check_close(w[b], total, (rel + (rep * T + 4) * 2.0 ** -23) * total.abs() + 1e-30)
        assert torch.equal(ck[b, :, m + c:], k0[b, :, m + c:]) and torch.equal(w[b, :, m + c:], w0[b, :, m + c:])


@pytest.mark.parametrize("T", [2, 40])
def test_weight_rows_past_the_capacity_are_not_stored(T):
    """Lengths on the device beyond what the cache holds: held to the capacity, nothing written past it."""
    G, cap, d = 2, 64, 64
    pad = torch.full((1, G + 1, cap, d), 7.0, dtype=BF16, device="cuda")
    q, k, v, ck0, cv0 = inputs(1, G, 2, T, cap, d, d, BF16, 41)
    big_k, big_v = pad.clone(), pad.clone()
    big_k[:, :G], big_v[:, :G] = ck0, cv0
    w = torch.full((1, G + 1, cap), 5.0, device="cuda")
    n = torch.tensor([cap - 1], dtype=torch.int32, device="cuda")
    log_kv_weight_attention(q, k, v, big_k[:, :G], big_v[:, :G], w[:, :G], n, 0.125)
    torch.cuda.synchronize()
    assert torch.equal(big_k[:, :G, cap - 1], k[:, :, 0]) and torch.equal(big_k[:, :G, :cap - 1], ck0[:, :, :cap - 1])
    assert bool((big_k[:, G] == 7.0).all()) and bool((big_v[:, G] == 7.0).all()) and bool((w[:, G] == 5.0).all())
    over = torch.tensor([cap + 1000], dtype=torch.int32, device="cuda")
    a = log_kv_tree_attention(q, k, v, ck0, cv0, over, torch.eye(T, dtype=torch.bool, device="cuda"), 0.125)
    b = log_kv_tree_attention(q, k, v, ck0, cv0, cap, torch.eye(T, dtype=torch.bool, device="cuda"), 0.125)
    assert torch.equal(a, b)
    under = torch.tensor([-3], dtype=torch.int32, device="cuda")
    a = log_kv_tree_attention(q, k, v, ck0, cv0, under, torch.eye(T, dtype=torch.bool, device="cuda"), 0.125)
    assert torch.equal(a, log_kv_tree_attention(q, k, v, ck0, cv0, 0, torch.eye(T, dtype=torch.bool, device="cuda"), 0.125))


def test_activation_dtypes_are_rounded_to_the_cache():
    q, k, v, ck, cv = inputs(1, 2, 2, 6, 50, 64, 64, torch.float32, 51)
    ck, cv = ck.to(BF16), cv.to(BF16)
    visible = tree_mask(6, 1).cuda()
    out = log_kv_tree_attention(q, k, v, ck, cv, 50, visible, 0.125)
    same = log_kv_tree_attention(q.to(BF16), k.to(BF16), v.to(BF16), ck, cv, 50, visible, 0.125)
    assert out.dtype == torch.float32 and torch.equal(out, same.float())


def test_rows_beyond_32_bit_offsets():
    """A cache whose last rows start past 2^32 bytes and 2^31 elements: zeros but for its last rows, whose logits stand out."""
    d, cap = 128, (1 << 24) + 37
    ck, cv = (torch.zeros(1, 1, cap, d, dtype=BF16, device="cuda") for _ in range(2))
    tail_k, tail_v = rows((1, 1, 5, d), BF16, 61, 4.0), rows((1, 1, 5, d), BF16, 62)
    ck[:, :, -5:], cv[:, :, -5:] = tail_k, tail_v
    q, k, v = rows((1, 2, 1, d), BF16, 63, 4.0), rows((1, 1, 1, d), BF16, 64), rows((1, 1, 1, d), BF16, 65)
    w = torch.zeros(1, 1, cap, device="cuda")
    out = log_kv_tree_attention(q, k, v, ck, cv, cap, torch.ones(1, 1, dtype=torch.bool, device="cuda"), 0.5)
    again = log_kv_weight_attention(q, k, v, ck, cv, w, torch.tensor([cap], dtype=torch.int32, device="cuda"), 0.5)
    assert torch.equal(out, again)
    for h in range(2):
        s = 0.5 * torch.cat((tail_k[0, 0], k[0, 0])).double().cpu() @ q[0, h, 0].double().cpu()
        top = max(float(s.max()), 0.0)
        p = torch.exp(s - top) / (torch.exp(s - top).sum() + (cap - 5) * math.exp(-top))
        vals = torch.cat((tail_v[0, 0], v[0, 0])).double().cpu()
        # half a step, and float32 sums over 2^24 equal terms in 64 x 4 shares of 2^16 rows (16384 additions a lane)
        err = 2.0 ** -8 * (p @ vals).abs() + (2.0 ** -10 + 2.0 ** -8) * (p @ vals.abs())
        check_close(out[0, h, 0], p @ vals, err)


def test_streams_and_another_current_device_stream():
    """Issued on a side stream behind the producer of its inputs: the result of the default stream."""
    q, k, v, ck, cv = inputs(2, 2, 2, 10, 3000, 128, 128, BF16, 71)
    visible = tree_mask(10, 3).cuda()
    want = log_kv_tree_attention(q, k, v, ck, cv, 3000, visible, 0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(ck)
        for _ in range(20):
            late.add_(0.0)
        late.copy_(ck)
        got = log_kv_tree_attention(q, k, v, late, cv, 3000, visible, 0.1)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("T,rep", [(1, 2), (30, 2), (100, 2)])
def test_captured_and_replayed(T, rep):
    """A captured step of tree attention and weight attention, replayed over changing inputs and lengths with eager
    calls between the replays: every replay equals the eager result."""
    G, cap, d = 2, 700, 64
    q, k, v, ck, cv = inputs(1, G, rep, T, cap, d, d, BF16, 81)
    w = torch.zeros(1, G, cap, device="cuda")
    n = torch.tensor([40], dtype=torch.int32, device="cuda")
    visible = tree_mask(T, 5).cuda()

    def step():
        a = log_kv_tree_attention(q, k, v, ck, cv, n, visible, 0.125)
        b = log_kv_weight_attention(q, k, v, ck, cv, w, n, 0.125)
        n.add_(T)
        return a, b

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    n.fill_(40)
    w.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = step()
    shadow = [x.clone() for x in (ck, cv, w, n)]
    for i in range(4):
        fresh = inputs(1, G, rep, T, cap, d, d, BF16, 90 + i)
        for x, y in zip((q, k, v), fresh):
            x.copy_(y)
        sk, sv, sw, sn = shadow
        want_a = log_kv_tree_attention(q, k, v, sk, sv, sn, visible, 0.125)
        want_b = log_kv_weight_attention(q, k, v, sk, sv, sw, sn, 0.125)
        sn.add_(T)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want_a) and torch.equal(b, want_b), i
        assert torch.equal(ck, sk) and torch.equal(cv, sv) and torch.equal(w, sw) and torch.equal(n, sn), i


@pytest.mark.parametrize("rep,T,dk,dv", [(2, 12, 128, 128), (1, 17, 96, 128), (4, 8, 80, 64)])
def test_17_to_32_queries_over_many_rows(rep, T, dk, dv):
    """Both operators where 17 to 32 queries take the tiled kernel: bf16, more than 64 features, a cache of many rows
    (in use: a few, and past a split's tiles)."""
    B, G, cap = 2, 1, 65600
    lengths = [4099, 33]
    q, k, v, ck, cv = inputs(B, G, rep, T, cap, dk, dv, BF16, 77)
    n, scale = torch.tensor(lengths, dtype=torch.int32, device="cuda"), dk ** -0.5
    visible = torch.stack([tree_mask(T, 60 + b, empty=(T - 1,)) for b in range(B)])
    want, _, bound, _ = reference(q, k, v, ck, cv, lengths, visible, scale)
    check_close(log_kv_tree_attention(q, k, v, ck, cv, n, visible.cuda(), scale), want, bound)
    causal = torch.ones(T, T, dtype=torch.bool).tril()[None].expand(B, T, T)
    want, column, bound, rel = reference(q, k, v, ck, cv, lengths, causal, scale)
    w = torch.rand(B, G, cap, generator=torch.Generator().manual_seed(8)).cuda()
    total = w.cpu().double()
    check_close(log_kv_weight_attention(q, k, v, ck, cv, w, n, scale), want, bound)
    for b, m in enumerate(lengths):
        total[b, :, :m] += column[b, :, :m]
        total[b, :, m:m + T] = column[b, :, cap:cap + T]
        check_close(w[b], total[b], (rel + (rep * T + 4) * 2.0 ** -23) * total[b].abs() + 1e-30)
        assert torch.equal(ck[b, :, m:m + T], k[b]) and torch.equal(cv[b, :, m:m + T], v[b])


@pytest.mark.parametrize("rep,T,d,dtype", [(2, 20, 64, BF16), (1, 70, 128, F16), (3, 61, 64, F16), (4, 70, 128, BF16)])
@pytest.mark.parametrize("lengths", [[4099, 33, 0, 700, 64], [5000, 5000, 4990, 5000, 5000], [1, 5000, 1, 1, 2],
                                     [-7, 2500, 9999, 1300, 640]])
def test_shares_by_length(lengths, rep, T, d, dtype):
    """Sequences of very different lengths in one call, whose rows are dealt out over the batch; the length of one
    call's sequence alone gives the same result but for the rounding of its shares' sums."""
    B, G, cap = len(lengths), 2, 5000
    q, k, v, ck, cv = inputs(B, G, rep, T, cap, d, d, dtype, 91)
    n, scale = torch.tensor(lengths, dtype=torch.int32, device="cuda"), d ** -0.5
    visible = torch.stack([tree_mask(T, 70 + b, empty=(T - 1,)) for b in range(B)])
    pick = [0, T // 2, T - 1]      # the reference's time goes by the queries: three tokens' rows of every head
    out = log_kv_tree_attention(q, k, v, ck, cv, n, visible.cuda(), scale)
    again = log_kv_tree_attention(q, k, v, ck, cv, n, visible.cuda(), scale)
    assert torch.equal(out, again)
    for b, m in enumerate(lengths):
        m = min(max(m, 0), cap)
        for t in pick:
            see = visible[b, t].nonzero().flatten().cuda()
            one = [x[b:b + 1] for x in (q[:, :, t:t + 1], torch.cat((ck[:, :, :m], k[:, :, see]), 2), torch.cat((cv[:, :, :m], v[:, :, see]), 2))]
            if one[1].size(2) == 0:
                assert bool((out[b, :, t] == 0).all())
                continue
            rows_k, rows_v = one[1], one[2]
            want, _, bound, _ = reference(one[0], rows_k[:, :, -1:], rows_v[:, :, -1:], rows_k[:, :, :-1], rows_v[:, :, :-1],
                                          [rows_k.size(2) - 1], torch.ones(1, 1, 1, dtype=torch.bool), scale)
            check_close(out[b:b + 1, :, t:t + 1], want, bound, f"row {b}, token {t}")


def test_shares_by_length_of_a_padded_batch_of_weights():
    B, G, rep, T, cap, d = 4, 2, 2, 40, 3000, 64
    lengths, counts = [2900, 0, 7, 1200], [T, 0, T - 1, 1]
    q, k, v, ck, cv = inputs(B, G, rep, T, cap, d, d, BF16, 92)
    w = torch.rand(B, G, cap, generator=torch.Generator().manual_seed(8)).cuda()
    total, before = w.cpu().double(), ck.clone()
    causal = torch.ones(T, T, dtype=torch.bool).tril()[None].expand(B, T, T)
    want, column, bound, rel = reference(q, k, v, ck, cv, lengths, causal, 0.125, counts=counts)
    out = log_kv_weight_attention(q, k, v, ck, cv, w, torch.tensor(lengths, device="cuda"), 0.125,
                                  counts=torch.tensor(counts, device="cuda"))
    check_close(out, want, bound)
    for b, (m, c) in enumerate(zip(lengths, counts)):
        total[b, :, :m] += column[b, :, :m]
        total[b, :, m:m + c] = column[b, :, cap:cap + c]
        check_close(w[b], total[b], (rel + (rep * T + 4) * 2.0 ** -23) * total[b].abs() + 1e-30)
        assert torch.equal(ck[b, :, m:m + c], k[b, :, :c]) and torch.equal(ck[b, :, m + c:], before[b, :, m + c:])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_wide_rows_of_many_queries_with_infinities(dtype):
    """Blocks of 32 queries of rows wider than 128 features; infinities and NaN reach only who sees them."""
    G, cap, rep, T, d = 1, 70, 4, 35, 256
    q, k, v, ck, cv = inputs(1, G, rep, T, cap, d, d, dtype, 21)
    visible = tree_mask(T, 2)
    v[0, 0, 1, 3], v[0, 0, 2, 200], v[0, 0, 4, 5] = math.inf, -math.inf, math.nan
    out = log_kv_tree_attention(q, k, v, ck, cv, 65, visible.cuda(), d ** -0.5)
    want, _, bound, _ = reference(q, k, v, ck, cv, [65], visible[None], d ** -0.5)
    assert bool(torch.isinf(want).any()) and bool(torch.isfinite(want[0, 0, 0]).all())
    check_close(out, want, bound)


def test_two_graphs_of_ragged_batches_at_once():
    """Two captured calls whose shares go by length, replayed on two streams together with an eager call on a third,
    over lengths that change between the replays."""
    B, G, rep, T, cap, d = 3, 2, 2, 24, 4000, 64
    sets = [inputs(B, G, rep, T, cap, d, d, BF16, 95 + i) for i in range(3)]
    ns = [torch.tensor([100, 4000, 1], dtype=torch.int32, device="cuda") for _ in sets]
    visible = tree_mask(T, 4).cuda()
    streams = [torch.cuda.Stream() for _ in sets]

    def call(i):
        q, k, v, ck, cv = sets[i]
        return log_kv_tree_attention(q, k, v, ck, cv, ns[i], visible, 0.125)

    call(0)
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    for lengths in ([100, 4000, 1], [4000, 4000, 4000], [3000, 0, 2222], [64, 65, 4000]):
        for n in ns:
            n.copy_(torch.tensor(lengths, dtype=torch.int32))
        want = [call(i) for i in range(3)]
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            eager = call(2)
        torch.cuda.synchronize()
        for got, w in zip((*outs, eager), want):
            assert torch.equal(got, w), lengths


def test_one_token_of_padded_rows():
    """A single token cut from rows of an odd width: the strides of its size-1 dimensions are odd too."""
    G, rep, d, cap = 2, 2, 64, 40
    wide = [rows((1, 1, h * d + 1), BF16, 50 + i)[..., 1:] for i, h in enumerate((G * rep, G, G))]
    q, k, v = (x.view(1, 1, h, d).transpose(1, 2) for x, h in zip(wide, (G * rep, G, G)))
    _, _, _, ck, cv = inputs(1, G, rep, 1, cap, d, d, BF16, 53)
    see = torch.ones(1, 1, dtype=torch.bool, device="cuda")
    out = log_kv_tree_attention(q, k, v, ck, cv, 37, see, 0.125)
    want, _, bound, _ = reference(q, k, v, ck, cv, [37], see.cpu()[None], 0.125)
    check_close(out, want, bound)
    dense = [torch.empty(x.shape, dtype=BF16, device="cuda").copy_(x) for x in (q, k, v)]
    assert torch.equal(out, log_kv_tree_attention(*dense, ck, cv, 37, see, 0.125))
    # Aligned rows with odd strides of dimensions of one element.
    odd = [x.as_strided(x.shape, (7, x.stride(1), 5, 1)) for x in dense]
    assert torch.equal(out, log_kv_tree_attention(*odd, ck, cv, 37, see, 0.125))
