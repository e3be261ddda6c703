"""Dual tensors (forward-mode derivatives) are refused where they would lose their tangent, whatever the mode of gradients
and before anything else is looked at (no GPU: no call gets as far as a launch)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from logkv_amd import (EvictingKVCache, PagedKVCache, SharedPrefix, log_kv_chunk_attention, log_kv_draft_attention, log_kv_evict,
                       log_kv_paged_append, log_kv_paged_attention, log_kv_prefix_attention, log_kv_rotary,
                       log_kv_slot_attention, log_kv_tree_attention, log_kv_weight_attention, pack_mid_kv)

B, H, G, T, D = 2, 4, 2, 3, 64


def rows(heads=G, tokens=T):
    return torch.zeros(B, heads, tokens, D)


Q, K, V = rows(H), rows(), rows()
PAGES, TABLE, TREE, BIAS = torch.zeros(8, G, 16, D), torch.zeros(B, 2, dtype=torch.int32), torch.ones(T, T).bool(), torch.zeros(B, G, T)
FREQ = torch.ones(D // 2)
CALLS = {
    "rotary": (lambda q, k, f: log_kv_rotary(q, k, f), (Q, K, FREQ)),
    "append": (lambda q, k, v, f: log_kv_paged_append(k, v, PAGES, PAGES, TABLE, 0, q=q, frequencies=f), (Q, K, V, FREQ)),
    "append's pages": (lambda a, b: log_kv_paged_append(K, V, a, b, TABLE, 0), (PAGES, PAGES)),
    "attention": (lambda q, k, v, a, b: log_kv_paged_attention(q, k, v, a, b, TABLE, 0, 1.0), (Q, K, V, PAGES, PAGES)),
    "prefix": (lambda k, v, b: log_kv_paged_attention(Q, K, V, PAGES, PAGES, TABLE, 0, 1.0, prefix=SharedPrefix(
        1, k=k, v=v, bias=b)), (K, V, BIAS)),
    "document": (lambda q, k, v, pk, pv: log_kv_prefix_attention(None, q, k, v, PAGES, PAGES, TABLE, 0, 1.0, pending=(pk, pv)),
                 (Q, K, V, K, V)),
    "paged cache": (lambda q, k, v: PagedKVCache(B, G, D, D, 8, scale=1.0, max_rows=16, device="cpu")(q, k, v), (Q, K, V)),
    "paged prefix": (lambda q, k, v: PagedKVCache(B, G, D, D, 8, scale=1.0, max_rows=16, device="cpu").prefix(q, k, v), (Q, K, V)),
    "paged draft": (lambda q, k, v: PagedKVCache(B, G, D, D, 8, scale=1.0, max_rows=16, device="cpu").draft(q, k, v, TREE), (Q, K, V)),
    "tree": (lambda q, k, v, a, b, c: log_kv_tree_attention(q, k, v, a, b, 0, TREE, 1.0, bias=c), (Q, K, V, K, V, BIAS)),
    "weights": (lambda q, k, v, a, b, w: log_kv_weight_attention(q, k, v, a, b, w, 0, 1.0), (Q, K, V, K, V, BIAS)),
    "evict": (lambda a, b, w: log_kv_evict(a, b, w, 1, 1), (K, V, BIAS)),
    "evicting cache": (lambda q, k, v: EvictingKVCache(B, G, D, D, 8, scale=1.0, device="cpu")(q, k, v), (Q, K, V)),
    "chunk": (lambda q, k, v: log_kv_chunk_attention(None, q, k, v, 1.0), (Q, K, V)),
    "draft": (lambda q, k, v, pk, pv: log_kv_draft_attention(None, q, k, v, TREE, 1.0, pending=(pk, pv)), (Q, K, V, K, V)),
    "slots": (lambda q, k, v, w: log_kv_slot_attention(q, k, v, w, 1.0), (Q, K, V, BIAS)),
    "pack": (lambda k, v: pack_mid_kv(None, None, k, v, 2 * D), (K, V)),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_a_tangent_is_refused(name, mode):
    call, args = CALLS[name]
    with forward_ad.dual_level(), mode():
        for i, x in enumerate(args):
            dual = list(args)
            dual[i] = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*dual)


def test_plain_tensors_at_a_dual_level_are_not():
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="device"):      # the next check
            log_kv_rotary(Q, None, FREQ)
        with pytest.raises(ValueError, match="device"):
            log_kv_paged_append(K.bfloat16(), V.bfloat16(), PAGES.bfloat16(), PAGES.bfloat16(), TABLE, 0)
