"""Caches, weights and eviction buffers whose dimensions of one element have strides of any size."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import EvictedRows, log_kv_evict, log_kv_tree_attention, log_kv_weight_attention
from row_reference import tree_mask
from test_gpu_row_attention import inputs

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def odd(x):
    """The same elements with odd strides of its dimensions of one element."""
    return x.as_strided(x.shape, [5 if n == 1 else s for n, s in zip(x.shape, x.stride())])


@pytest.mark.parametrize("B,G,T,cap", [(1, 2, 3, 40), (2, 1, 3, 40), (1, 1, 1, 40), (1, 1, 1, 1), (2, 2, 1, 1)])
def test_attention(B, G, T, cap):
    q, k, v, ck, cv = inputs(B, G, 2, T, cap, 64, 64, BF16, 11)
    see = tree_mask(T, 2).cuda()
    n = torch.tensor([cap - T if cap > 1 else 0] * B, dtype=torch.int32, device="cuda")
    want = log_kv_tree_attention(q, k, v, ck, cv, n, see, 0.125)
    assert torch.equal(log_kv_tree_attention(odd(q), odd(k), odd(v), odd(ck), odd(cv), n, odd(see), 0.125), want)
    w = torch.rand(B, G, cap, device="cuda")
    plain, other = [x.clone() for x in (ck, cv, w)], [odd(x.clone()) for x in (ck, cv, w)]
    want = log_kv_weight_attention(q, k, v, *plain, n, 0.125)
    assert torch.equal(log_kv_weight_attention(odd(q), odd(k), odd(v), *other, n, 0.125), want)
    assert all(torch.equal(x, y) for x, y in zip(plain, other))


@pytest.mark.parametrize("B,G,cap,keep", [(1, 2, 40, 7), (2, 1, 40, 1), (1, 1, 1, 1), (1, 1, 50, 20)])
def test_eviction(B, G, cap, keep):
    _, _, _, ck, cv = inputs(B, G, 1, 1, cap, 64, 64, BF16, 12)
    w = torch.rand(B, G, cap, device="cuda")
    pos = torch.arange(cap, device="cuda").expand(B, G, cap).contiguous()
    want = log_kv_evict(ck, cv, w, cap, keep, positions=pos)
    got = log_kv_evict(odd(ck), odd(cv), odd(w), cap, keep, positions=odd(pos))
    out = EvictedRows(*(odd(torch.empty_like(x)) if x.ndim > 2 and i < 4 else torch.empty_like(x) for i, x in enumerate(want)))
    log_kv_evict(odd(ck), odd(cv), odd(w), cap, keep, positions=odd(pos), out=out)
    for a, b, c in zip(want, got, out):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_other_strides_are_still_refused():
    q, k, v, ck, cv = inputs(1, 2, 2, 3, 40, 64, 64, BF16, 13)
    see = tree_mask(3, 2).cuda()
    wide = torch.zeros(1, 2, 40, 68, dtype=BF16, device="cuda")[..., :64]
    with pytest.raises(ValueError, match="16-byte aligned"):
        log_kv_tree_attention(q, k, v, wide, cv, 40, see, 0.125)
    w = torch.rand(1, 2, 80, device="cuda")[:, :, ::2]
    with pytest.raises(ValueError, match="contiguous"):
        log_kv_weight_attention(q, k, v, ck, cv, w, 37, 0.125)
    with pytest.raises(ValueError, match="contiguous"):
        log_kv_evict(ck, cv, w, 40, 8)
    with pytest.raises(ValueError, match="16-byte aligned"):
        log_kv_evict(wide, cv, torch.rand(1, 2, 40, device="cuda"), 40, 8)
