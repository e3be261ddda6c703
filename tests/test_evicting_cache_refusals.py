"""A refused call of an EvictingKVCache leaves it as it was, also where the call would have evicted first (no GPU: no call
gets as far as a launch)."""

from __future__ import annotations

import math

import pytest
import torch

from logkv_amd import EvictingKVCache

B, G, D, DV = 2, 2, 64, 32


def rows(heads, tokens, d, **kw):
    return torch.zeros(B, heads, tokens, d, dtype=kw.pop("dtype", torch.bfloat16), **kw)


@pytest.fixture
def full(monkeypatch):
    """A cache whose next call has to evict."""
    cache = EvictingKVCache(B, G, D, DV, 8, scale=0.125, device="cpu")
    cache._bound = cache.capacity

    def evict():
        raise AssertionError("rows were dropped for a call that is refused")

    monkeypatch.setattr(cache, "evict", evict)
    return cache


BAD = {
    "values' width": lambda T: (rows(4, T, D), rows(G, T, D), rows(G, T, D)),
    "keys' width": lambda T: (rows(4, T, D), rows(G, T, DV), rows(G, T, DV)),
    "queries' width": lambda T: (rows(4, T, DV), rows(G, T, D), rows(G, T, DV)),
    "queries' heads": lambda T: (rows(3, T, D), rows(G, T, D), rows(G, T, DV)),
    "no heads": lambda T: (rows(0, T, D), rows(G, T, D), rows(G, T, DV)),
    "groups": lambda T: (rows(4, T, D), rows(1, T, D), rows(1, T, DV)),
    "more values": lambda T: (rows(4, T, D), rows(G, T, D), rows(G, T + 1, DV)),
    "fewer values": lambda T: (rows(4, T + 1, D), rows(G, T + 1, D), rows(G, T, DV)),
    "more keys": lambda T: (rows(4, T, D), rows(G, T + 1, D), rows(G, T, DV)),
    "batch": lambda T: (rows(4, T, D)[:1], rows(G, T, D), rows(G, T, DV)),
    "3-dimensional": lambda T: (rows(4, T, D)[0], rows(G, T, D), rows(G, T, DV)),
    "1-dimensional": lambda T: (rows(4, T, D).flatten(), rows(G, T, D), rows(G, T, DV)),
    "device": lambda T: (rows(4, T, D), rows(G, T, D), rows(G, T, DV, device="meta")),
    "counts' shape": lambda T: (rows(4, T, D), rows(G, T, D), rows(G, T, DV), torch.ones(3, dtype=torch.int32)),
    "counts' dtype": lambda T: (rows(4, T, D), rows(G, T, D), rows(G, T, DV), torch.ones(B)),
}


@pytest.mark.parametrize("tokens", [1, 2, 7])     # 7: more than a block
@pytest.mark.parametrize("bad", BAD)
def test_a_refused_call_drops_no_rows(full, bad, tokens):
    before = [None if x is None else x.clone() for x in full._rows]
    with pytest.raises(ValueError):
        full(*BAD[bad](tokens))
    assert full._bound == full.capacity
    assert all(x is None or torch.equal(x, y) for x, y in zip(full._rows, before))


def test_a_refused_dtype_drops_no_rows(full):
    with pytest.raises(NotImplementedError):
        full(rows(4, 1, D), rows(G, 1, D, dtype=torch.float64), rows(G, 1, DV))
    with pytest.raises(ValueError, match="2.19"):
        full(rows((1 << 20) * G, 1, 8)[..., :1].expand(-1, -1, -1, D), rows(G, 1, D), rows(G, 1, DV))


@pytest.mark.parametrize("args,kw", [
    ((2, 2, 60, 64, 8), {}), ((2, 2, 64, 12, 8), {}), ((2, 2, 264, 64, 8), {}), ((2, 2, 64, 512, 8), {}),
    ((300, 300, 64, 64, 8), {}), ((2, 2, 64, 64, 8), {"scale": 0.0}), ((2, 2, 64, 64, 8), {"scale": math.nan}),
    ((2, 2, 64, 64, 8), {"scale": math.inf}), ((2, 2, 64, 64, 8), {"dtype": torch.float32})])
def test_sizes_that_no_call_takes_are_refused_at_construction(args, kw):
    with pytest.raises(ValueError):
        EvictingKVCache(*args, device="meta", **{"scale": 0.125, **kw})
