"""Eviction by accumulated weight on the device: the rows that stay, exactly."""

from __future__ import annotations

import math

import pytest
import torch

from logkv_amd import EvictedRows, log_kv_evict
from row_reference import evict_reference

pytestmark = pytest.mark.gpu


def check(ck, cv, w, lengths, keep, recent, got, positions=None):
    B, G, cap = w.shape
    wh = w.cpu()
    for b in range(B):
        n = min(max(lengths[b], 0), cap)
        assert int(got.lengths[b]) == min(n, keep)
        for g in range(G):
            idx = evict_reference(wh[b, g], n, keep, recent)
            m = len(idx)
            assert got.kept[b, g].tolist() == idx + [-1] * (keep - m), (b, g)
            at = torch.tensor(idx, dtype=torch.long, device=ck.device)
            for x, y in ((got.k, ck), (got.v, cv), (got.weights, w)):
                kept = x[b, g, :keep]
                assert torch.equal(kept[:m].view(torch.uint8), y[b, g][at].view(torch.uint8))
                assert bool((kept[m:] == 0).all())
            if positions is not None:
                assert torch.equal(got.positions[b, g, :m], positions[b, g][at])
                assert bool((got.positions[b, g, m:keep] == -1).all())


CASES = [
    # B, G, cap, lengths, keep, recent
    (1, 1, 2, [2], 1, 0), (1, 1, 2, [2], 1, 1), (1, 2, 1, [1], 1, 0), (1, 2, 5, [0], 3, 1),
    (2, 2, 100, [100, 37], 40, 10), (2, 2, 100, [41, 40], 40, 40), (1, 3, 1088, [1088], 1024, 256),
    (3, 1, 1025, [1025, 1024, 0], 1024, 0), (1, 2, 5000, [4999], 100, 99), (1, 2, 8200, [8193], 4096, 7),
    (1, 1, 32768, [32768], 4096, 512), (1, 1, 40000, [39999], 39998, 1), (1, 1, 70001, [70001], 5, 2),
]


@pytest.mark.parametrize("values", ["heavy", "ties", "odd"])
@pytest.mark.parametrize("B,G,cap,lengths,keep,recent", CASES)
def test_evict(B, G, cap, lengths, keep, recent, values):
    g = torch.Generator().manual_seed(cap + keep)
    d = 8
    ck, cv = (torch.randn(B, G, cap, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    w = torch.exp(2 * torch.randn(B, G, cap, generator=g))
    if values == "ties":
        w = torch.randint(0, 3, (B, G, cap), generator=g).float()
    elif values == "odd":
        pick = torch.randint(0, 8, (B, G, cap), generator=g)
        special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, -1.5, 1e-42, 2.0])
        w = torch.where(torch.rand(B, G, cap, generator=g) < 0.7, special[pick], w)
    w = w.cuda()
    pos = torch.randint(0, 1 << 40, (B, G, cap), generator=g).cuda()
    got = log_kv_evict(ck, cv, w, torch.tensor(lengths, dtype=torch.int32, device="cuda"), keep, recent=recent, positions=pos)
    check(ck, cv, w, lengths, keep, recent, got, pos)


@pytest.mark.parametrize("dtype,dk,dv", [(torch.float16, 64, 128), (torch.float32, 4, 20), (torch.uint8, 16, 48),
                                         (torch.bfloat16, 256, 8)])
def test_types_and_strides(dtype, dk, dv):
    B, G, cap, keep = 2, 3, 90, 50
    size = torch.empty(0, dtype=dtype).element_size()
    pad = 16 // size
    ck, cv = ((torch.rand(B, cap, G, d + pad, device="cuda") * 100).to(dtype)[..., :d].transpose(1, 2) for d in (dk, dv))
    w = torch.rand(B, G, 2 * cap, device="cuda")[..., cap:]
    got = log_kv_evict(ck, cv, w, 90, keep, recent=3)
    assert got.positions is None
    check(ck, cv, w, [90, 90], keep, 3, got)


def test_into_a_second_buffer_set():
    """Buffers of more rows than are kept: the first `keep` rows are written, the rest stays."""
    B, G, cap, keep, d = 2, 2, 80, 30, 64
    ck, cv = (torch.randn(B, G, cap, d, device="cuda").to(torch.bfloat16) for _ in range(2))
    w, pos = torch.rand(B, G, cap, device="cuda"), torch.arange(cap, device="cuda").expand(B, G, cap).contiguous()
    out = EvictedRows(torch.full_like(ck, 7.0), torch.full_like(cv, 7.0), torch.full_like(w, 7.0), torch.full_like(pos, 7),
                      torch.empty(B, G, keep, dtype=torch.int32, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda"))
    lengths = torch.tensor([80, 20], dtype=torch.int32, device="cuda")
    got = log_kv_evict(ck, cv, w, lengths, keep, recent=8, positions=pos, out=out)
    assert got is out
    check(ck, cv, w, [80, 20], keep, 8, got, pos)
    for t in out[:4]:
        assert bool((t[:, :, keep:] == 7).all())
    with pytest.raises(ValueError, match="overlap"):
        log_kv_evict(ck, cv, w, lengths, keep, positions=pos, out=out._replace(k=ck))
    with pytest.raises(ValueError, match="overlap"):
        log_kv_evict(ck, cv, w, lengths, keep, positions=pos, out=out._replace(v=out.k))
    with pytest.raises(ValueError, match="match the cache"):
        log_kv_evict(ck, cv, w, lengths, keep, positions=pos, out=out._replace(kept=out.kept[:, :, :-1]))


def test_rows_beyond_32_bit_offsets():
    d, cap = 128, (1 << 24) + 5
    ck, cv = (torch.zeros(1, 1, cap, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ck[0, 0, -1], ck[0, 0, -3], cv[0, 0, -3] = 3.0, 5.0, 6.0
    w = torch.zeros(1, 1, cap, device="cuda")
    w[0, 0, cap - 3] = 1.0
    got = log_kv_evict(ck, cv, w, cap, 4, recent=1)
    assert got.kept[0, 0].tolist() == [0, 1, cap - 3, cap - 1]
    assert bool((got.k[0, 0, 2] == 5.0).all()) and bool((got.v[0, 0, 2] == 6.0).all()) and bool((got.k[0, 0, 3] == 3.0).all())


def test_captured_and_replayed():
    B, G, cap, keep, d = 2, 2, 600, 128, 64
    ck, cv = (torch.randn(B, G, cap, d, device="cuda").to(torch.bfloat16) for _ in range(2))
    w = torch.rand(B, G, cap, device="cuda")
    lengths = torch.tensor([600, 300], dtype=torch.int32, device="cuda")
    log_kv_evict(ck, cv, w, lengths, keep, recent=16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = log_kv_evict(ck, cv, w, lengths, keep, recent=16)
    for i in range(4):
        w.copy_(torch.rand(B, G, cap, device="cuda"))
        lengths.copy_(torch.tensor([600 - 77 * i, 300 - 90 * i], dtype=torch.int32))
        want = log_kv_evict(ck, cv, w, lengths, keep, recent=16)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert a is None or torch.equal(a, b), i
