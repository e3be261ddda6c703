"""A call of a PagedKVCache that fails behind its checks (memory that runs out, a launch that is refused) leaves the cache as
it was, and the same or a smaller call can follow (no GPU: the launches are stand-ins)."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import paged_cache
from test_paged_cache_refusals import B, D, DV, G, new, rows, same, state


@pytest.fixture
def launches(monkeypatch):
    """Stand-ins for the launches; raise the error of the one that ``fails`` names."""
    fails = {}

    def launch(name, give):
        def call(*args, **kw):
            if name in fails:
                raise fails[name]
            return give(*args, **kw)
        monkeypatch.setattr(paged_cache, name, call)

    launch("log_kv_paged_append", lambda k, v, *a, q=None, **kw: (q, k))
    launch("log_kv_paged_attention", lambda q, k, v, *a, **kw: q.new_zeros(*q.shape[:3], v.size(3)))
    return fails


def call(cache, n, batch=B, of="__call__", **kw):
    return getattr(cache, of)(rows(batch, 4, n, D), rows(batch, G, n, D), rows(batch, G, n, DV), **kw)


@pytest.mark.parametrize("at", ["log_kv_paged_append", "log_kv_paged_attention"])
@pytest.mark.parametrize("error", [torch.cuda.OutOfMemoryError("no memory"), ValueError("too many blocks")], ids=["memory", "refused"])
def test_prefixes(launches, at, error):
    cache = new(pages=16)
    for held in (0, 10):       # without a prefix, and behind the first block of one
        if held:
            call(cache, held, 2, "prefix")
        before = state(cache)
        launches[at] = error
        with pytest.raises(type(error)):
            call(cache, 70, 2, "prefix")
        assert same(state(cache), before) and (cache._prefix_table.size(1) == 1 if held else cache._prefix_table is None)
        del launches[at]
    assert call(cache, 3, 2, "prefix").shape == (2, 4, 3, DV)      # fewer tokens, a narrower table
    assert cache.prefix_rows == 2 * 13 and cache.free_pages == 14
    launches[at] = error
    with pytest.raises(type(error)):
        call(cache, 1)
    del launches[at]
    call(cache, 5, 2, "prefix")       # no sequence has a row yet
    assert cache.prefix_rows == 2 * 18 and cache.free_pages == 12


@pytest.mark.parametrize("at", ["log_kv_paged_append", "log_kv_paged_attention"])
def test_steps(launches, at):
    cache = new(pages=16)
    call(cache, 10)
    before = state(cache)
    for error in (torch.cuda.OutOfMemoryError("no memory"), ValueError("too many blocks")):
        launches[at] = error
        for kw in ({}, dict(counts=torch.tensor([30, 0, 1, 30], dtype=torch.int32))):
            with pytest.raises(type(error)):
                call(cache, 30, **kw)
            assert same(state(cache), before)
    del launches[at]
    upload, cache._upload = cache._upload, None      # the table's own update fails
    with pytest.raises(TypeError):
        call(cache, 30)
    cache._upload = upload
    assert same(state(cache), before)
    call(cache, 20)
    assert cache.lengths.tolist() == [30] * B and cache.free_pages == 8
    lines = sum(cache._pages, [])
    assert len(set(lines)) == 8 and not set(lines) & set(cache._free)
    assert all(cache.table[b, :2].tolist() == cache._pages[b] for b in range(B)) and (cache.table[:, 2:] == -1).all()


@pytest.mark.parametrize("name", ["free", "trim", "reset", "some"])
def test_pages_are_not_taken_back_in_a_capture(launches, monkeypatch, name):
    """The host would hand the pages out again at once, the device forget them at a replay."""
    cache = new(pages=16)
    call(cache, 4, 2, "prefix")
    call(cache, 20)
    before, pages = state(cache), cache.k_pages
    cache.k_pages = pages.view(pages.shape).as_subclass(OnDevice)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        cache.free([1]) if name == "some" else getattr(cache, name)()
    cache.k_pages = pages
    assert same(state(cache), before)


class OnDevice(torch.Tensor):
    is_cuda = True


def test_frequencies_that_every_call_would_refuse():
    for frequencies, kind in ((torch.ones(4, dtype=torch.int64), ValueError), (torch.ones(4, dtype=torch.bfloat16), ValueError),
                              (torch.ones(4, requires_grad=True), NotImplementedError)):
        with pytest.raises(kind, match="frequencies"):
            new(frequencies=frequencies)
    assert new(frequencies=torch.ones(4)).frequencies.dtype == torch.float32


def test_padded_batches_are_told_of_trim(launches):
    """Padding counts until trim(), which the errors name; after it the calls go on."""
    cache = new(pages=16)
    counts = torch.tensor([1, 0, 2, 1], dtype=torch.int32)
    for _ in range(4):
        call(cache, 16, counts=counts)
    with pytest.raises(RuntimeError, match=r"trim\(\)"):      # 64 of 64 rows may be in use
        call(cache, 1)
    cache.trim()
    assert cache.lengths.tolist() == [4, 0, 8, 4] and cache.free_pages == 13
    call(cache, 16)
    cache = new(pages=4)
    call(cache, 16, counts=counts)
    with pytest.raises(RuntimeError, match=r"trim\(\)"):
        call(cache, 16, counts=counts)
    cache.trim()
    call(cache, 1, counts=counts)


def test_sequences_to_free_are_indices(launches):
    """A mask's truth values were taken for the indices 0 and 1, numbers with a fraction for those below."""
    cache = new(pages=16)
    call(cache, 20)
    before = state(cache)
    mask = [False, False, True, False]
    for bad in (mask, torch.tensor(mask), [1.5], torch.tensor([1.0]), [[1]], [torch.tensor(True)], [-1], ["1"]):
        with pytest.raises(ValueError, match="indices"):
            cache.free(bad)
    assert same(state(cache), before)
    for some, left in ((torch.tensor([2]), [20, 20, 0, 20]), ((0, torch.tensor(2)), [0, 20, 0, 20]), (torch.tensor(3), [0, 20, 0, 0]),
                       ((), [0, 20, 0, 0]), (iter([1]), [0] * B)):
        cache.free(some)
        assert cache.lengths.tolist() == cache._bound == left
    assert cache.free_pages == 16
