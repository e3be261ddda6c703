"""Which documents a PagedKVCache takes as its sequences' prefix (no GPU: nothing is attended)."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import LogKVStreamingAttention, LogStructuredKVCache
from test_paged_cache_refusals import D, DV, G, new, rows, same, state


def document(**over):
    """A cache's attributes that sharing looks at."""
    doc = LogStructuredKVCache.__new__(LogStructuredKVCache)
    doc.__dict__.update(dict(batch_size=2, n_groups=G, k_dim=D, v_dim=DV, token_count=40, semantic_pack_backend="auto",
                             recent_k=torch.zeros(2, G, 4, D)), **over)
    return doc


def test_a_document():
    cache = new()
    cache.share(document())
    assert cache._first == 40 and cache._sharing() == 2
    cache.reset()
    engine = LogKVStreamingAttention.__new__(LogKVStreamingAttention)
    engine.cache = document()
    engine._log_kv_pending = (torch.zeros(2, G, 1, D), torch.zeros(2, G, 1, DV))
    cache.share(engine)
    assert cache._first == 41


def test_beside_another():
    """A second document took the first one's place without a word."""
    cache = new()
    cache.share(document())
    before = state(cache)
    with pytest.raises(RuntimeError, match="beside no other"):
        cache.share(document(token_count=7))
    with pytest.raises(RuntimeError, match="beside no other"):
        cache.prefix(rows(2, 4, 1, D), rows(2, G, 1, D), rows(2, G, 1, DV))
    assert same(state(cache), before)


@pytest.mark.parametrize("over", [
    dict(batch_size=3), dict(n_groups=1), dict(k_dim=32), dict(v_dim=D),
    # What every later call would refuse:
    dict(recent_k=torch.zeros(2, G, 4, D, device="meta")), dict(semantic_pack_backend="torch")], ids=lambda x: next(iter(x)))
def test_others(over):
    cache = new()
    before = state(cache)
    with pytest.raises((ValueError, NotImplementedError)):
        cache.share(document(**over))
    assert same(state(cache), before)
    with pytest.raises(ValueError):
        new(dtype=torch.float16).share(document())
