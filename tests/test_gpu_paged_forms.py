"""Every form that the two passes of a paged attention take together, with shares of many tiles, against attention in 64
bits under row_reference's bounds. Which form a call takes follows its sizes; the plan that the library reports is checked,
so that another rule cannot take a form out of these tests in silence."""

from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from logkv_amd import SharedPrefix, _paged, log_kv_paged_attention
from row_reference import check_close, tree_mask

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
PAGE = 16

# d, B, H, G, T, most own rows, prefixes, most prefix rows, then the plan: the own pass's waves of 32 queries (tiled) or
# columns of 16 (streamed), the prefixes' likewise.
FORMS = [
    (64, 48, 8, 8, 1, 1000, 1, 1500, (0, 2, 2, 0)),
    (64, 48, 8, 8, 2, 1000, 2, 700, (0, 2, 2, 0)),
    (64, 24, 32, 8, 9, 300, 2, 700, (2, 0, 2, 0)),
    (64, 48, 8, 8, 2, 1000, 1, 6000, (0, 2, 4, 0)),
    (64, 48, 8, 8, 3, 1000, 2, 3000, (0, 2, 4, 0)),
    (64, 6, 16, 4, 70, 300, 2, 700, (4, 0, 4, 0)),
    (64, 48, 32, 8, 3, 300, 1, 700, (0, 2, 8, 0)),
    (64, 48, 32, 8, 2, 300, 2, 1500, (0, 2, 8, 0)),
    (64, 8, 16, 8, 70, 300, 4, 700, (8, 0, 8, 0)),
    (128, 24, 8, 8, 2, 992, 1, 6000, (0, 1, 2, 0)),
    (128, 48, 8, 8, 1, 1000, 2, 3000, (0, 1, 2, 0)),
    (128, 24, 32, 8, 9, 300, 3, 700, (2, 0, 2, 0)),
    (128, 64, 8, 8, 1, 1000, 2, 1500, (0, 1, 4, 0)),
    (128, 12, 8, 8, 70, 64, 3, 700, (4, 0, 4, 0)),
    (128, 48, 16, 8, 3, 1000, 2, 700, (0, 1, 8, 0)),
    (128, 16, 8, 8, 70, 64, 4, 700, (8, 0, 8, 0)),
    # Without a prefix.
    (64, 8, 32, 8, 9, 1000, 0, 0, (2, 0, 0, 0)),
    (64, 2, 8, 8, 70, 4000, 0, 0, (4, 0, 0, 0)),
    (64, 4, 8, 8, 300, 300, 0, 0, (8, 0, 0, 0)),
    (128, 8, 32, 8, 9, 1000, 0, 0, (2, 0, 0, 0)),
    (128, 2, 8, 8, 70, 4000, 0, 0, (4, 0, 0, 0)),
    (128, 4, 8, 8, 300, 300, 0, 0, (8, 0, 0, 0)),
]


def randn(seed, *shape, dtype=BF16, factor=1.0):
    return (factor * torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")).to(dtype)


def plan(B, H, G, T, d, table_len, N, prefix_len, paged, page=PAGE):
    args = _paged.PagedArgs(n_batch=B, n_heads=H, n_groups=G, tq=T, dk=d, dv=d, page=page, table_len=table_len, n_prefixes=N,
                            prefix_len=prefix_len, prefix_table=1 if paged else None)
    out = (C.c_int32 * 8)()
    assert _paged.paged_lib().logkv_paged_plan(C.byref(args), out) == 0
    return list(out)


def in_pages(G, d, lengths, dtype, seed):
    """(k pages, v pages, table) of random rows."""
    width = max(1, -(-max(lengths) // PAGE))
    order = torch.randperm(len(lengths) * width, generator=torch.Generator().manual_seed(seed)).int().view(len(lengths), width)
    return (*(randn(seed + i, order.numel(), G, PAGE, d, dtype=dtype) for i in (1, 2)), order.cuda())


def rows_of(pages, line, n):
    """Rows ``[G, n, d]`` of a sequence, in 64 bits."""
    x = pages[line.long()[:-(-n // PAGE)]].transpose(0, 1)
    return x.reshape(x.size(0), -1, x.size(3))[:, :n].double()


def want_of(q, keys, vals, add, see, scale, half):
    """(out, bound) of queries ``[rep, T, d]`` over rows ``[n, d]`` with logits' addends ``[n]`` and a mask ``[T, n]``."""
    rep, T, d = q.shape
    x = q.double().view(rep * T, d)
    see = see[None].expand(rep, -1, -1).reshape(rep * T, -1)
    s = (x @ keys.t() * scale + add).masked_fill(~see, -math.inf)
    empty = ~see.any(dim=1)
    p = torch.softmax(s.masked_fill(empty[:, None], 0.0), dim=1).masked_fill(empty[:, None] | ~see, 0.0)
    out = p @ vals
    size = (scale * (x.abs() @ keys.abs().t()) + add.abs().nan_to_num(posinf=0.0)).masked_fill(p == 0.0, 0.0).amax(dim=1, keepdim=True)
    e = (d + 8) * 2.0 ** -24 * size
    parts = 2.0 ** -14 if half == 2.0 ** -8 else 2.0 ** -21
    factor = 2 * (2 * e + 2.0 ** -20) + parts + (see.sum(dim=1, keepdim=True) + 8) * 2.0 ** -24
    bound = half * out.abs() + (1 + half) * factor * (p @ vals.abs()) + (2.0 ** -24 if half == 2.0 ** -11 else 2.0 ** -25)
    return out.view(rep, T, -1), bound.view(rep, T, -1)


VARIANTS = [("pages", BF16), ("pages", F16), ("float bias", BF16), ("half bias", F16), ("rows", BF16)]


@pytest.mark.parametrize("form,rows,dtype", [(f, *x) for f in FORMS for x in VARIANTS if f[6] or x[0] != "half bias"],
                         ids=lambda x: "-".join(map(str, x[:8])) if isinstance(x, tuple) else str(x).replace("torch.", ""))
def test_forms(form, rows, dtype):
    d, B, H, G, T, own, N, most, forms = form
    rep, scale, half = H // G, d ** -0.5, 2.0 ** -8 if dtype == BF16 else 2.0 ** -11
    lengths = [own - (97 * b) % own for b in range(B)]      # (without a prefix: "float bias" stands for trees, "rows" for counts)
    sizes = [most, most // 3, 0, most - 5][:N]
    q, k, v = randn(1, B, H, T, d, dtype=dtype, factor=2.0), randn(2, B, G, T, d, dtype=dtype), randn(3, B, G, T, d, dtype=dtype)
    kp, vp, table = in_pages(G, d, lengths + (sizes if rows == "pages" else []), dtype, 4)
    line, prefix, bias = table[:B, :-(-own // PAGE)].contiguous(), None, None
    if N:
        pn = torch.tensor(sizes, dtype=torch.int32, device="cuda")
        if rows == "pages":
            tables = table[B:, :-(-most // PAGE)].contiguous()
            prefix = SharedPrefix(pn, table=tables)
            shared = [(rows_of(kp, tables[i], n), rows_of(vp, tables[i], n)) for i, n in enumerate(sizes)]
        else:
            pk, pv = randn(5, N, G, most, d, dtype=dtype), randn(6, N, G, most, d, dtype=dtype)
            if rows != "rows":
                bias = randn(7, N, G, most, dtype=torch.float32 if rows == "float bias" else dtype)
                bias[:, :, 3::11] = -math.inf
            prefix = SharedPrefix(pn, k=pk, v=pv, bias=bias, bias_scale=0.5)
            shared = [(pk[i, :, :n].double(), pv[i, :, :n].double()) for i, n in enumerate(sizes)]
    # The form: its kernels, several tiles a share, and shares by length where prefixes differ.
    p = plan(B, H, G, T, d, line.size(1), N, -(-most // PAGE) if rows == "pages" else most, rows == "pages")
    assert (p[0], p[1], p[4], p[5]) == forms
    tiles, shares, room = (-(-most // 64), *p[6:]) if N else (-(-own // 64) + -(-T // 64), *p[2:4])
    assert tiles // shares >= 5 and (N < 2 or shares == 1 or room > shares)
    kw = {}
    see = torch.ones(T, T, dtype=torch.bool).tril().cuda().expand(B, T, T)
    if rows == "float bias":
        kw["visible"] = see = torch.stack([tree_mask(T, b, empty=(T - 1,) if b % 2 else ()) for b in range(B)]).cuda()
    elif rows == "rows":
        counts = [max(0, T - b % (T + 2)) for b in range(B)]
        kw["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        see = see & (torch.arange(T, device="cuda") < kw["counts"][:, None])[:, None]
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = log_kv_paged_attention(q, k, v, kp, vp, line, n, scale, prefix=prefix, **kw)
    assert torch.equal(out, log_kv_paged_attention(q, k, v, kp, vp, line, n, scale, prefix=prefix, **kw))
    wants, bounds = torch.zeros(out.shape, dtype=torch.float64), torch.zeros(out.shape, dtype=torch.float64)
    for b in range(B):
        i = b // (B // N) if N else 0
        m = sizes[i] if N else 0
        own_k, own_v = rows_of(kp, line[b], lengths[b]), rows_of(vp, line[b], lengths[b])
        for g in range(G):
            keys, vals = [own_k[g], k[b, g].double()], [own_v[g], v[b, g].double()]
            add = torch.zeros(m + lengths[b] + T, dtype=torch.float64, device="cuda")
            if N:
                keys.insert(0, shared[i][0][g]), vals.insert(0, shared[i][1][g])
                if bias is not None:
                    add[:m] = bias[i, g, :m].double() * 0.5
            mask = torch.cat((torch.ones(T, m + lengths[b], dtype=torch.bool, device="cuda"), see[b]), dim=1) & (add != -math.inf)
            if "counts" in kw:
                mask &= torch.arange(T, device="cuda")[:, None] < kw["counts"][b]
            heads = slice(g * rep, (g + 1) * rep)
            wants[b, heads], bounds[b, heads] = want_of(q[b, heads], torch.cat(keys), torch.cat(vals), add, mask, scale, half)
    check_close(out, wants, bounds, p)


def test_an_infinity_in_every_form():
    """A row's infinity in a later tile of a share reaches every query that sees the row, in tiled and streamed passes."""
    for d, B, H, G, T, own, N, most, forms in FORMS:
        kp, vp, table = in_pages(G, d, [own] * B + [most] * N, BF16, 8)
        line = table[:B, :-(-own // PAGE)].contiguous()
        prefix = SharedPrefix(most, table=table[B:, :-(-most // PAGE)].contiguous()) if N else None
        q, k, v = randn(1, B, H, T, d, factor=2.0), randn(2, B, G, T, d), randn(3, B, G, T, d)
        clean = log_kv_paged_attention(q, k, v, kp, vp, line, own, d ** -0.5, prefix=prefix)
        assert torch.isfinite(clean).all()
        want = clean.clone()
        vp[line[B - 1, own // 2 // PAGE].long(), :, own // 2 % PAGE, d - 1] = -math.inf
        want[B - 1, :, :, d - 1] = -math.inf
        if N:
            at = most * 2 // 3
            vp[prefix.table[0, at // PAGE].long(), G - 1, at % PAGE, 5] = math.inf
            want[:B // N, (G - 1) * H // G:, :, 5] = math.inf
        got = log_kv_paged_attention(q, k, v, kp, vp, line, own, d ** -0.5, prefix=prefix)
        assert torch.equal(got, want), (forms, T, N)


@pytest.mark.parametrize("B,T,forms", [(2, 1, (0, 1, 0, 1)), (16, 20, (4, 0, 4, 0)), (8, 40, (8, 0, 8, 0))],
                         ids=["streamed", "tiled", "wide blocks"])
def test_pages_beyond_2_31_elements(B, T, forms):
    """K's and V's pages whose offsets pass 31 and 32 bits, in both passes by both kernels."""
    H, G, d, page, pages = 32, 8, 128, 256, 16500      # 4.3e9 elements
    assert pages * G * page * d > 2 ** 32
    p = plan(B, H, G, T, d, 4, 2, 4, True, page)
    assert (p[0], p[1], p[4], p[5]) == forms
    pools = [torch.empty(pages, G, page, d, dtype=BF16, device="cuda") for _ in range(2)]
    used = [pages - 1 - i for i in range(2 * B + 4)] + [pages // 2 + i for i in range(2 * B + 4)]      # beyond 2^32 and 2^31
    for i, x in enumerate(pools):
        for j, at in enumerate(used):
            x[at] = randn(100 * i + j, G, page, d)
    line = torch.tensor(used, dtype=torch.int32, device="cuda").view(2, -1).t().reshape(-1, 4).contiguous()      # [B + 2, 4]
    q, k, v = randn(1, B, H, T, d, factor=2.0), randn(2, B, G, T, d), randn(3, B, G, T, d)
    few = [x[line.flatten().long()].clone() for x in pools]
    near = torch.arange(line.numel(), dtype=torch.int32, device="cuda").view(-1, 4)
    n = torch.tensor([1000 - 7 * b for b in range(B)], dtype=torch.int32, device="cuda")
    got, want = (log_kv_paged_attention(q, k, v, kp, vp, at[:B], n, d ** -0.5, prefix=SharedPrefix(1000, table=at[B:]))
                 for (kp, vp), at in ((pools, line), (few, near)))
    assert torch.isfinite(want).all() and torch.equal(got, want)


@pytest.mark.parametrize("B,H,tiled", [(2, 4, False), (32, 4, True)], ids=["streamed", "tiled"])
def test_contiguous_rows_beyond_2_31_elements(B, H, tiled):
    """A prefix of contiguous rows: rows of one group beyond 2^31 elements from its first, the second group's beyond 2^32."""
    G, T, d, cap, last = 2, 1, 128, 17_000_000, 300
    assert (cap - last) * d > 2 ** 31 and (2 * cap - last) * d > 2 ** 32
    p = plan(B, H, G, T, d, 1, 1, cap, False)
    assert (p[4] > 0) == tiled
    pk, pv = (torch.zeros(1, G, cap, d, dtype=BF16, device="cuda") for _ in range(2))
    bias = torch.full((1, G, cap), -math.inf, device="cuda")
    bias[:, :, -last:] = randn(9, G, last, dtype=torch.float32)
    pk[:, :, -last:], pv[:, :, -last:] = randn(5, G, last, d), randn(6, G, last, d)
    pv[:, :, :5] = math.nan      # hidden
    q, k, v = randn(1, B, H, T, d, factor=2.0), randn(2, B, G, T, d), randn(3, B, G, T, d)
    kp, vp, table = in_pages(G, d, [5] * B, BF16, 4)
    out = log_kv_paged_attention(q, k, v, kp, vp, table, 5, d ** -0.5, prefix=SharedPrefix(cap, k=pk, v=pv, bias=bias))
    for b in range(B):
        own_k, own_v = rows_of(kp, table[b], 5), rows_of(vp, table[b], 5)
        for g in range(G):
            keys, vals = (torch.cat((x[0, g, -last:].double(), y[g], z[b, g].double())) for x, y, z in ((pk, own_k, k), (pv, own_v, v)))
            add = torch.cat((bias[0, g, -last:].double(), torch.zeros(6, dtype=torch.float64, device="cuda")))
            heads = slice(g * H // G, (g + 1) * H // G)
            want, bound = want_of(q[b, heads], keys, vals, add, torch.ones(T, last + 6, dtype=torch.bool, device="cuda"), d ** -0.5, 2.0 ** -8)
            check_close(out[b, heads], want.cpu(), bound.cpu(), (b, g))
