"""A refused call of a PagedKVCache leaves it as it was (no GPU: no call gets as far as a launch)."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import PagedKVCache

B, G, D, DV = 4, 2, 64, 32


def rows(batch, heads, tokens, d, dtype=torch.bfloat16):
    return torch.zeros(batch, heads, tokens, d, dtype=dtype)


def new(**kw):
    return PagedKVCache(B, G, D, DV, kw.pop("pages", 8), **{**dict(scale=0.125, max_rows=64, page_size=16, device="cpu"), **kw})


def state(cache):
    return ([list(x) for x in cache._pages], sorted(cache._free), list(cache._bound), cache.lengths.clone(), cache.table.clone(),
            [list(x) for x in cache._prefix_pages], cache._prefix_rows, cache._first, cache._compressed)


def same(a, b):
    return all(torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(a, b))


BAD = {
    "values' width": lambda T: (rows(B, 4, T, D), rows(B, G, T, D), rows(B, G, T, D)),
    "keys' width": lambda T: (rows(B, 4, T, D), rows(B, G, T, DV), rows(B, G, T, DV)),
    "queries' width": lambda T: (rows(B, 4, T, DV), rows(B, G, T, D), rows(B, G, T, DV)),
    "queries' heads": lambda T: (rows(B, 3, T, D), rows(B, G, T, D), rows(B, G, T, DV)),
    "no heads": lambda T: (rows(B, 0, T, D), rows(B, G, T, D), rows(B, G, T, DV)),
    "groups": lambda T: (rows(B, 4, T, D), rows(B, 1, T, D), rows(B, 1, T, DV)),
    "more values": lambda T: (rows(B, 4, T, D), rows(B, G, T, D), rows(B, G, T + 1, DV)),
    "batch": lambda T: (rows(B + 1, 4, T, D), rows(B + 1, G, T, D), rows(B + 1, G, T, DV)),
    "dtypes": lambda T: (rows(B, 4, T, D), rows(B, G, T, D, torch.float16), rows(B, G, T, DV)),
    "no tokens": lambda T: (rows(B, 4, 0, D), rows(B, G, 0, D), rows(B, G, 0, DV)),
    "dimensions": lambda T: (rows(B, 4, T, D)[0], rows(B, G, T, D), rows(B, G, T, DV)),
}


@pytest.mark.parametrize("what", BAD)
@pytest.mark.parametrize("T", [1, 20])
def test_bad_rows(what, T):
    cache = new()
    before = state(cache)
    with pytest.raises(ValueError):
        cache(*BAD[what](T))
    with pytest.raises(ValueError):
        cache.draft(*BAD[what](T), torch.ones(T, T, dtype=torch.bool))
    with pytest.raises(ValueError):      # as prefixes, of which five do not divide the batch
        cache.prefix(*BAD[what](T))
    assert same(state(cache), before)


def test_other_dtypes_counts_and_positions():
    cache = new(frequencies=torch.ones(4, dtype=torch.float64))
    before = state(cache)
    good = rows(B, 4, 1, D), rows(B, G, 1, D), rows(B, G, 1, DV)
    with pytest.raises(NotImplementedError):
        cache(*(x.double() for x in good))
    for counts in (torch.zeros(3, dtype=torch.int32), torch.zeros(B), torch.zeros(B, 1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            cache(*good, counts=counts)
    with pytest.raises(ValueError, match="positions"):
        cache.draft(*good, torch.ones(1, 1, dtype=torch.bool))
    assert same(state(cache), before)


def test_too_few_pages_and_too_many_rows():
    cache = new(pages=7)
    before = state(cache)
    with pytest.raises(RuntimeError, match="pages left"):
        cache(rows(B, 4, 17, D), rows(B, G, 17, D), rows(B, G, 17, DV))      # two pages for each of four
    with pytest.raises(RuntimeError, match="at most 64 rows"):
        cache(rows(B, 4, 65, D), rows(B, G, 65, D), rows(B, G, 65, DV))
    with pytest.raises(RuntimeError, match="pages left"):
        cache.prefix(rows(2, 4, 60, D), rows(2, G, 60, D), rows(2, G, 60, DV))
    assert same(state(cache), before) and cache.free_pages == 7


def test_prefixes_come_first_and_alone():
    cache = new()
    cache._bound[1] = 3
    q, k, v = rows(2, 4, 1, D), rows(2, G, 1, D), rows(2, G, 1, DV)
    with pytest.raises(RuntimeError, match="before"):
        cache.prefix(q, k, v)
    with pytest.raises(ValueError, match="document"):
        cache.share(object())
    cache._bound[1] = 0
    for n in (3, 8):
        with pytest.raises(ValueError, match="divide"):
            cache.prefix(rows(n, 4, 1, D), rows(n, G, 1, D), rows(n, G, 1, DV))


def test_pages_are_handed_out_and_taken_back():
    cache = new()
    cache._reserve(cache._pages, cache.table, [17, 1, 0, 16])
    assert [len(x) for x in cache._pages] == [2, 1, 0, 1] and cache.free_pages == 4
    used = sum(cache._pages, [])
    assert len(set(used)) == 4 and not set(used) & set(cache._free)
    for b, line in enumerate(cache._pages):
        assert cache.table[b].tolist() == line + [-1] * (4 - len(line))
    cache._bound = [17, 1, 0, 16]
    cache.lengths.copy_(torch.tensor([3, 1, 0, 16]))
    cache.trim()
    assert [len(x) for x in cache._pages] == [1, 1, 0, 1] and cache._bound == [3, 1, 0, 16] and cache.free_pages == 5
    assert cache.table[0].tolist() == cache._pages[0] + [-1] * 3
    cache.free([0, 3, 0])
    assert cache.free_pages == 7 and cache._bound == [0, 1, 0, 0] and cache.lengths.tolist() == [0, 1, 0, 0]
    with pytest.raises(ValueError):
        cache.free([4])
    cache.reset()
    assert cache.free_pages == 8 and sorted(cache._free) == list(range(8)) and (cache.table == -1).all()


@pytest.mark.parametrize("over", [
    dict(pages=0), dict(max_rows=0), dict(page_size=8), dict(page_size=24), dict(scale=0.0), dict(scale=float("nan")),
    dict(amplitude=float("inf")), dict(dtype=torch.float32), dict(max_rows=2 ** 31), dict(frequencies=torch.ones(33)),
    dict(frequencies=torch.ones(2, 2))])
def test_construction(over):
    with pytest.raises(ValueError):
        new(**over)


def test_construction_widths():
    for widths in ((60, 64), (64, 264), (0, 64), (64, 4)):
        with pytest.raises(ValueError):
            PagedKVCache(1, 1, *widths, 4, scale=1.0, max_rows=16, device="cpu")


def test_the_limit_of_queries_is_of_sequences_that_share_rows():
    """2^19 query rows a KV group for the sequences behind one prefix; each sequence has its own without one."""
    T = 1 << 15      # 8 heads a group: half of the limit a sequence, twice the limit all four

    def large(batch):
        one = torch.zeros((), dtype=torch.bfloat16)
        return one.expand(batch, 8 * G, T, D), one.expand(batch, G, T, D), one.expand(batch, G, T, DV)

    cache = new(max_rows=T)
    for call in (cache, cache.prefix):
        with pytest.raises(RuntimeError, match="pages left"):      # not refused before
            call(*large(B))
    cache._prefix_pages = [[], []]
    with pytest.raises(RuntimeError, match="pages left"):
        cache(*large(B))
    cache._prefix_pages = [[]]
    with pytest.raises(ValueError, match="split the call"):
        cache(*large(B))
    cache._prefix_pages = []
    with pytest.raises(ValueError, match="split the call"):
        cache(*(x.expand(B, -1, 4 * T, -1) for x in (y[:, :, :1] for y in large(B))))
