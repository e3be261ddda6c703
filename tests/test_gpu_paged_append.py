"""Appends to a paged cache on the GPU, with and without the rotation, against the formula in 64 bits."""

import pytest
import torch

from paged_reference import inverse, pool, rotate, within

pytestmark = pytest.mark.gpu


def make(B, H, T, d, dtype, seed):
    return torch.randn(B, H, T, d, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def expected(before, rows, bounds, table, lengths, counts, page):
    """Pages after the append (64 bits) with the bound of each value: rows kept as they were have none."""
    want, bound = before.detach().cpu().double(), torch.zeros(before.shape, dtype=torch.float64)
    table = table.cpu()
    for b, n in enumerate(lengths):
        for t in range(counts[b]):
            at = n + t
            if not 0 <= at < table.size(1) * page:
                continue
            p = int(table[b, at // page])
            if 0 <= p < want.size(0):
                want[p, :, at % page], bound[p, :, at % page] = rows[b, :, t], bounds[b, :, t]
    return want, bound


def plain(x, to):
    return x.detach().cpu().to(to).double(), torch.zeros(x.shape, dtype=torch.float64)


CASES = [
    # B, H, G, T, dk, dv, r, page, lengths
    (1, 4, 2, 1, 128, 128, 128, 16, [0]),
    (3, 4, 4, 1, 64, 64, 32, 64, [15, 16, 200]),
    (2, 3, 1, 37, 80, 96, 20, 16, [5, 48]),
    (4, 2, 2, 5, 192, 128, 64, 32, [31, 0, 27, 33]),
    (2, 2, 1, 9, 7, 3, 4, 16, [3, 14]),
    (2, 1, 1, 3, 256, 64, 256, 256, [255, 1]),
    (64, 2, 1, 40, 64, 64, 64, 16, [3 * b for b in range(64)]),
]


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:8])))
def test_rotated_append(case, interleaved, dtype, cache):
    from logkv_amd import log_kv_paged_append

    B, H, G, T, dk, dv, r, page, lengths = case
    for variant in range(3):
        q, k, v = make(B, H, T, dk, dtype, 1), make(B, G, T, dk, dtype, 2), make(B, G, T, dv, dtype, 3)
        if variant == 1:
            q, k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))
        counts = [T] * B if variant == 0 else [max(0, T - b) for b in range(B)]
        kp, vp, table = pool(B, G, dk, dv, page, [n + T for n in lengths], cache, 4, "cuda")
        f = inverse(10000.0, r // 2)
        n_dev = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        pos = torch.tensor(lengths)[:, None] + torch.arange(T)
        extra = {}
        if variant == 0:
            extra["first"], pos = 1000, pos + 1000
        elif variant == 1:
            first = torch.arange(B) * 77
            extra["first"], pos = first.cuda(), pos + first[:, None]
        else:
            pos = torch.randint(0, 1 << 20, (B, T), generator=torch.Generator().manual_seed(9))
            extra["positions"] = pos.cuda()
        if variant:
            extra["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        before = kp.clone(), vp.clone()
        q_out, k_out = log_kv_paged_append(k, v, kp, vp, table, n_dev, q=q, frequencies=f.cuda(), interleaved=interleaved,
                                           amplitude=1.25, **extra)
        assert q_out.dtype == dtype and k_out.dtype == cache
        within(q_out, *rotate(q, f, pos, interleaved, 1.25), "queries")
        want, bound = rotate(k, f, pos, interleaved, 1.25, to=cache)
        within(k_out, want, bound, "keys")
        within(kp, *expected(before[0], want, bound, table, lengths, counts, page), "key pages")
        within(vp, *expected(before[1], *plain(v, cache), table, lengths, counts, page), "value pages")
        # What is stored is what is returned, bit for bit.
        at = lengths[0]
        if counts[0]:
            assert torch.equal(kp[table[0, at // page].item(), :, at % page], k_out[0, :, 0])


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16)])
def test_without_a_rotation(dtype, cache):
    from logkv_amd import log_kv_paged_append

    B, G, T, dk, dv, page = 2, 2, 21, 64, 32, 16
    k, v, q = make(B, G, T, dk, dtype, 1), make(B, G, T, dv, dtype, 2), make(B, 4, T, dk, dtype, 3)
    kp, vp, table = pool(B, G, dk, dv, page, [T + 7] * B, cache, 4, "cuda")
    before = kp.clone(), vp.clone()
    q_out, k_out = log_kv_paged_append(k, v, kp, vp, table, 7, q=q)
    assert q_out is q and (k_out is k if dtype == cache else torch.equal(k_out, k.to(cache)))
    within(kp, *expected(before[0], *plain(k, cache), table, [7, 7], [T, T], page))
    within(vp, *expected(before[1], *plain(v, cache), table, [7, 7], [T, T], page))
    assert log_kv_paged_append(k, v, kp, vp, table, 7)[0] is None


def test_rows_without_a_page_are_not_stored():
    """Entries outside the pool, rows behind the table's last, negative lengths: nothing else changes."""
    from logkv_amd import log_kv_paged_append

    B, G, T, d, page = 6, 1, 20, 32, 16
    k, v = make(B, G, T, d, torch.bfloat16, 1), make(B, G, T, d, torch.bfloat16, 2)
    kp, vp, _ = pool(1, G, d, d, page, [16 * 7], torch.bfloat16, 3, "cuda", spare=0)
    table = torch.tensor([[0, -1], [7, 1], [2, 2 ** 31 - 1], [3, 4], [5, 6], [-2 ** 31, 7]], dtype=torch.int32, device="cuda")
    lengths = [3, 3, 3, 25, -10, 0]
    before = kp.clone(), vp.clone()
    f = inverse(10000.0, 16)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    _, k_out = log_kv_paged_append(k, v, kp, vp, table, n, frequencies=f.cuda())
    pos = torch.tensor(lengths)[:, None] + torch.arange(T)
    want, bound = rotate(k, f, pos)
    within(k_out, want, bound)
    within(kp, *expected(before[0], want, bound, table, lengths, [T] * B, page))
    within(vp, *expected(before[1], *plain(v, v.dtype), table, lengths, [T] * B, page))
    # An empty pool or an empty table: the rotation alone.
    for kp0, vp0, t0 in ((kp[:0], vp[:0], table), (kp, vp, table[:, :0])):
        keep = kp.clone()
        _, again = log_kv_paged_append(k, v, kp0, vp0, t0, n, frequencies=f.cuda())
        assert torch.equal(again, k_out) and torch.equal(kp, keep)


def test_strided_pools():
    """Pages of one buffer that holds keys beside values, and of a pool with tokens before heads."""
    from logkv_amd import log_kv_paged_append

    B, G, T, d, page = 2, 3, 5, 64, 16
    k, v = make(B, G, T, d, torch.float16, 1), make(B, G, T, d, torch.float16, 2)
    table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32, device="cuda")
    both = torch.zeros(5, 2, page, G, d, dtype=torch.float16, device="cuda")
    kp, vp = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    f = inverse(10000.0, 32)
    _, k_out = log_kv_paged_append(k, v, kp, vp, table, 14, frequencies=f.cuda())
    want, bound = rotate(k, f, (torch.arange(T) + 14).expand(B, T))
    within(kp, *expected(torch.zeros_like(kp), want, bound, table, [14, 14], [T, T], page))
    within(vp, *expected(torch.zeros_like(vp), *plain(v, v.dtype), table, [14, 14], [T, T], page))
    # Rows that are not 16-byte aligned.
    odd = torch.zeros(4 * G * page * d + 1, dtype=torch.float16, device="cuda")[1:].view(4, G, page, d)
    vp2 = torch.zeros(4, G, page, d, dtype=torch.float16, device="cuda")
    log_kv_paged_append(k, v, odd, vp2, table, 14, frequencies=f.cuda())
    within(odd, *expected(torch.zeros_like(odd), want, bound, table, [14, 14], [T, T], page))


def test_far_pages():
    """Page offsets beyond 2^31 elements."""
    from logkv_amd import log_kv_paged_append

    G, d, page, pages = 8, 128, 256, 8200 + 100
    kp = torch.zeros(pages, G, page, d, dtype=torch.bfloat16, device="cuda")      # 2.18e9 elements
    vp = torch.zeros(pages, G, page, 8, dtype=torch.bfloat16, device="cuda")
    k, v = make(1, G, 3, d, torch.bfloat16, 1), make(1, G, 3, 8, torch.bfloat16, 2)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    log_kv_paged_append(k, v, kp, vp, table, 255)
    assert torch.equal(kp[pages - 1, :, 255], k[0, :, 0]) and torch.equal(kp[pages - 2, :, :2], k[0, :, 1:])
    assert torch.equal(vp[pages - 2, :, :2], v[0, :, 1:])
    assert int(torch.count_nonzero(kp[: pages - 2].view(torch.int16).view(-1, page * d).amax(dim=1))) == 0


def test_captured_and_on_a_side_stream():
    from logkv_amd import log_kv_paged_append

    B, G, d, page = 2, 2, 64, 16
    f = inverse(10000.0, 32).cuda()
    q, k, v = (make(B, n, 1, d, torch.bfloat16, n) for n in (4, G, G + 1))
    v = v[:, :G].contiguous()
    kp, vp, table = pool(B, G, d, d, page, [64, 64], torch.bfloat16, 4, "cuda")
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    log_kv_paged_append(k, v, kp, vp, table, lengths, q=q, frequencies=f)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = log_kv_paged_append(k, v, kp, vp, table, lengths, q=q, frequencies=f)
        graphs.append((graph, out))
    for step in range(5):
        k.normal_(generator=torch.Generator("cuda").manual_seed(step)), lengths.add_(7)
        kp2, vp2 = kp.clone(), vp.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = log_kv_paged_append(k, v, kp2, vp2, table, lengths, q=q, frequencies=f)
        torch.cuda.current_stream().wait_stream(side)
        graph, out = graphs[step % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kp, kp2) and torch.equal(vp, vp2) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    from logkv_amd import log_kv_paged_append

    k, v, q = make(2, 2, 3, 64, torch.bfloat16, 1), make(2, 2, 3, 64, torch.bfloat16, 2), make(2, 4, 3, 64, torch.bfloat16, 3)
    kp, vp, table = pool(2, 2, 64, 64, 16, [32, 32], torch.bfloat16, 4, "cuda")
    before = kp.clone(), vp.clone()
    f = inverse(10000.0, 32).cuda()
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    good = dict(k=k, v=v, k_pages=kp, v_pages=vp, table=table, lengths=n, q=q, frequencies=f)
    for change, kind in (
            (dict(k=k[0]), ValueError), (dict(v=v[:, :, :2]), ValueError), (dict(q=q[:, :, :1]), ValueError),
            (dict(k=k.float()), ValueError), (dict(k=k.cpu()), ValueError), (dict(k_pages=kp[:, :1]), ValueError),
            (dict(v_pages=vp.half()), ValueError), (dict(k_pages=kp.float(), v_pages=vp.float()), ValueError),
            (dict(k_pages=kp[:, :, :8], v_pages=vp[:, :, :8]), ValueError), (dict(table=table.long()), ValueError),
            (dict(table=table[:1]), ValueError), (dict(table=table.cpu()), ValueError), (dict(lengths=30), ValueError),
            (dict(lengths=-1), ValueError), (dict(lengths=n[:1]), ValueError), (dict(lengths=n.float()), ValueError),
            (dict(frequencies=torch.cat((f, f))), ValueError), (dict(frequencies=f.cpu()), ValueError),
            (dict(first=1.5), TypeError), (dict(first=n), ValueError), (dict(positions=3), ValueError),
            (dict(positions=torch.zeros(2, 4, dtype=torch.int64, device="cuda")), ValueError),
            (dict(counts=n[:1]), ValueError), (dict(counts=n.float()), ValueError), (dict(amplitude=float("nan")), ValueError),
            (dict(k_pages=kp[:1].expand(4, -1, -1, -1), v_pages=vp[:1].expand(4, -1, -1, -1)), ValueError),
            (dict(k_pages=kp.transpose(2, 3).contiguous().transpose(2, 3)), ValueError),
            (dict(k=k.clone().requires_grad_()), NotImplementedError), (dict(k=k.double(), v=v.double(), q=q.double()), NotImplementedError)):
        with pytest.raises(kind):
            log_kv_paged_append(**{**good, **change})
    torch.cuda.synchronize()
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])
