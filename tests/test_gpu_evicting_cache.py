"""An exact cache of a fixed budget as it is used: prefill, decode, drafts and evictions in turn, every output and
weight against the 64-bit form of the rows that are there and every eviction exactly."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import EvictingKVCache
from row_reference import check_close, evict_reference, reference, tree_mask

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def rows(shape, dtype, g):
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def checked_evict(cache, ordinals):
    """Evicts and compares with the rows' own weights; the ordinals of the rows that stay."""
    w, k, v = cache.weights.cpu(), cache.k.clone(), cache.v.clone()
    lengths = cache.lengths.tolist()
    kept = cache.evict()
    out = []
    for b, n in enumerate(lengths):
        out.append([])
        for h in range(cache.n_groups):
            idx = evict_reference(w[b, h], n, cache.budget, cache.recent)
            assert kept[b, h].tolist() == idx + [-1] * (cache.budget - len(idx))
            assert torch.equal(cache.k[b, h, :len(idx)], k[b, h, idx]) and torch.equal(cache.v[b, h, :len(idx)], v[b, h, idx])
            assert torch.equal(cache.weights[b, h, :len(idx)].cpu(), w[b, h, idx])
            out[-1].append([ordinals[b][h][i] for i in idx])
    return out


@pytest.mark.parametrize("dtype,dk,dv,rep,budget,recent,block", [
    (BF16, 64, 64, 2, 40, 8, 16), (F16, 128, 64, 1, 33, 0, 7), (BF16, 32, 16, 4, 5, 5, 1), (BF16, 128, 128, 4, 100, 25, 50)])
def test_attend_evict_draft_and_accept(dtype, dk, dv, rep, budget, recent, block):
    B, G = 2, 2
    scale = dk ** -0.5
    g = torch.Generator().manual_seed(budget)
    cache = EvictingKVCache(B, G, dk, dv, budget, scale=scale, recent=recent, block=block, dtype=dtype, track_positions=True)
    twin = EvictingKVCache(B, G, dk, dv, budget, scale=scale, recent=recent, block=block, dtype=dtype)
    ordinals, seen, evictions = [[[] for _ in range(G)] for _ in range(B)], [0] * B, 0
    bound = 0

    def step(q, k, v, counts):
        nonlocal ordinals, evictions, bound
        T = q.size(2)
        if bound + T > cache.capacity:
            ordinals = checked_evict(cache, ordinals)
            evictions += 1
            bound = min(bound, budget)
        bound += T
        n, w0 = cache.lengths.tolist(), cache.weights.cpu().double()
        causal = torch.ones(T, T, dtype=torch.bool).tril()[None].expand(B, T, T)
        want, column, err, rel = reference(q, k, v, cache.k.clone(), cache.v.clone(), n, causal, scale, counts=counts)
        on_device = None if counts is None else torch.tensor(counts, device="cuda")
        out = cache(q, k, v, counts=on_device)
        check_close(out, want, err)
        assert torch.equal(out, twin(q, k, v, counts=on_device))   # which evicts by itself
        cap = cache.capacity
        for b, m in enumerate(n):
            c = T if counts is None else counts[b]
            assert int(cache.lengths[b]) == m + c
            total = w0[b, :, :m + c].clone()
            total[:, m:] = 0
            total += column[b][:, list(range(m)) + list(range(cap, cap + c))]
            check_close(cache.weights[b, :, :m + c], total, (rel + (rep * T + 4) * 2.0 ** -23) * total.abs() + 1e-30)
            assert torch.equal(cache.k[b, :, m:m + c], k[b, :, :c]) and torch.equal(cache.v[b, :, m:m + c], v[b, :, :c])
            for h in range(G):
                ordinals[b][h] += range(seen[b], seen[b] + c)
                assert cache.positions[b, h, :m + c].tolist() == ordinals[b][h]
            seen[b] += c
        return out

    for i in range(14):
        T = min(block, (block, 1, 1, 2, max(1, block // 2))[i % 5])     # a call of one block: no eviction inside it
        q, k, v = rows((B, G * rep, T, dk), dtype, g), rows((B, G, T, dk), dtype, g), rows((B, G, T, dv), dtype, g)
        step(q, k, v, None if i % 3 else [T, T // 2])
        if i % 4 == 3:      # a draft, of which the first path is committed
            n = 6
            q, k, v = rows((B, G * rep, n, dk), dtype, g), rows((B, G, n, dk), dtype, g), rows((B, G, n, dv), dtype, g)
            visible = tree_mask(n, i)
            want, _, err, _ = reference(q, k, v, cache.k, cache.v, cache.lengths.tolist(), visible[None].expand(B, n, n), scale)
            before = cache.k.clone(), cache.weights.clone(), cache.lengths.clone()
            check_close(cache.draft(q, k, v, visible.cuda()), want, err)
            assert all(torch.equal(x, y) for x, y in zip(before, (cache.k, cache.weights, cache.lengths)))
            path = [j for j in range(n) if visible[n - 1, j]][:block]
            step(q[:, :, path], k[:, :, path], v[:, :, path], None)
    assert evictions > 1
    for name in ("lengths", "weights", "k", "v"):
        for b in range(B):
            m = int(cache.lengths[b])
            x, y = getattr(cache, name)[b], getattr(twin, name)[b]
            assert torch.equal(x, y) if name == "lengths" else torch.equal(x[:, :m], y[:, :m])


def test_a_long_call_is_its_blocks():
    B, G, d, block, T = 1, 2, 64, 16, 75
    g = torch.Generator().manual_seed(4)
    q, k, v = rows((B, 4, T, d), BF16, g), rows((B, G, T, d), BF16, g), rows((B, G, T, d), BF16, g)
    whole, parts = (EvictingKVCache(B, G, d, d, 24, scale=0.125, block=block) for _ in range(2))
    out = whole(q, k, v, counts=torch.tensor([70], device="cuda"))
    for a in range(0, T, block):
        b = min(T, a + block)
        y = parts(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], counts=torch.tensor([max(0, min(70, b) - a)], device="cuda"))
        assert torch.equal(out[:, :, a:b], y)
    assert torch.equal(whole.weights, parts.weights) and torch.equal(whole.lengths, parts.lengths)
    whole.reset()
    fresh = EvictingKVCache(B, G, d, d, 24, scale=0.125, block=block)
    assert torch.equal(whole(q[:, :, :9], k[:, :, :9], v[:, :, :9]), fresh(q[:, :, :9], k[:, :, :9], v[:, :, :9]))


def test_refusals():
    cache = EvictingKVCache(2, 2, 64, 64, 8, scale=0.125)
    q, k = torch.zeros(2, 4, 1, 64, dtype=BF16, device="cuda"), torch.zeros(2, 2, 1, 64, dtype=BF16, device="cuda")
    for bad in (lambda: cache(q[:, :, :0], k[:, :, :0], k[:, :, :0]), lambda: cache(q[:1], k[:1], k[:1]),
                lambda: cache(q, k, k[..., :32]), lambda: cache(q, k, k, counts=torch.tensor([1, 1])),
                lambda: cache(q, k, k, counts=torch.ones(2, device="cuda")), lambda: cache(q[:, :3], k, k)):
        with pytest.raises(ValueError):
            bad()
    assert cache.lengths.tolist() == [0, 0]
    cache(q, k, k)
    see = torch.ones(1, 1, dtype=torch.bool, device="cuda")
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            for call in (lambda: cache(q, k, k), cache.evict, lambda: cache.draft(q, k, k, see)):
                with pytest.raises(RuntimeError, match="captured"):
                    call()
            q.add_(0)
        finally:
            graph.capture_end()
    assert cache.lengths.tolist() == [1, 1]
