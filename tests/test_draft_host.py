"""Host logic of drafts and of the evicting cache that needs no device: accepted paths, positions, refused sizes."""

import pytest
import torch

from logkv_amd import EvictingKVCache, LogKVStreamingAttention
from logkv_amd.streaming import _check_path, _join_pos, _pick


def test_paths():
    assert _check_path([], 4, 2) == [[]] and _check_path(torch.zeros(0, dtype=torch.long), 4, 2) == [[]]
    assert _check_path([0, 2, 3], 4, 2) == [[0, 2, 3]] and _check_path(torch.tensor([1]), 4, 2) == [[1]]
    assert _check_path([[0, 1], (2, 3)], 4, 2) == [[0, 1], [2, 3]] and _check_path(torch.tensor(3), 4, 2) == [[3]]
    for bad in ([4], [-1], [1, 0], [2, 2], [[0], [1], [2]], [[0], [1, 2]], torch.tensor([[3, 4]])):
        with pytest.raises(ValueError, match="path"):
            _check_path(bad, 4, 2)


def test_picked_rows():
    x = torch.arange(2 * 3 * 4 * 5).view(2, 3, 4, 5)
    assert torch.equal(_pick(x, torch.tensor([[1, 3]])), x[:, :, [1, 3]])
    got = _pick(x, torch.tensor([[0, 2], [1, 3]]))
    assert torch.equal(got[0], x[0][:, [0, 2]]) and torch.equal(got[1], x[1][:, [1, 3]])


def test_joined_positions():
    one, two = torch.tensor([3]), torch.tensor([[4, 5], [7, 8]])
    assert _join_pos(None, one) is None and _join_pos(one, None) is None
    assert _join_pos(one, one).tolist() == [3, 3]
    assert _join_pos(one, two).tolist() == [[3, 4, 5], [3, 7, 8]] and _join_pos(two, one).tolist() == [[4, 5, 3], [7, 8, 3]]


class Recorder:
    """A cache that only records what is committed."""

    semantic_clusters, alpha_exact_tokens, recent_size = True, 0, 4

    def __init__(self):
        self.commits = []

    def add_recent(self, k, v, *, k_raw, input_pos, span_ends):
        assert k.shape == v.shape == k_raw.shape
        self.commits.append((k[0, 0, :, 0].tolist(), None if input_pos is None else input_pos.tolist(), span_ends))


@pytest.mark.parametrize("path,commits,left", [
    ([0], [[9, 0]], None), ([1, 3], [[9, 1]], 3), ([0, 1, 2, 3, 4, 5], [[9, 0], [1, 2, 3, 4]], 5), ([], [], 9)])
def test_accept_keeps_the_commit_boundaries(path, commits, left):
    cache = Recorder()
    engine = LogKVStreamingAttention(cache, 0.125)
    row = lambda *x: torch.tensor(x, dtype=torch.float32).view(1, 1, -1, 1)  # noqa: E731
    engine._log_kv_pending = (row(9), row(9), row(9), torch.tensor([9]), None)
    k = row(0, 1, 2, 3, 4, 5)
    engine._drafted = (k, k, k, torch.arange(6), None)
    engine.accept(path)
    assert [c[0] for c in cache.commits] == commits and [c[1] for c in cache.commits] == commits
    pending = engine._log_kv_pending
    assert (pending is None) if left is None else (pending[0].flatten().tolist() == [left] and pending[3].tolist() == [left])
    with pytest.raises(RuntimeError, match="draft"):
        engine.accept([0])


def test_evicting_cache_sizes():
    for over in ({"budget": 0}, {"block": 0}, {"recent": 9}, {"recent": -1}, {"dtype": torch.float32}, {"n_groups": 0}):
        args = {"batch_size": 1, "n_groups": 1, "k_dim": 8, "v_dim": 8, "budget": 8, "scale": 1.0, "device": "cpu", **over}
        with pytest.raises(ValueError):
            EvictingKVCache(**args)
    cache = EvictingKVCache(1, 2, 8, 16, 8, scale=1.0, device="cpu", track_positions=True)
    assert cache.k.shape == (1, 2, 10, 8) and cache.v.shape == (1, 2, 10, 16) and cache.positions.shape == (1, 2, 10)
    assert (cache.recent, cache.block, cache.capacity, cache.lengths.tolist()) == (2, 2, 10, [0])
    x = torch.zeros(1, 2, 1, 8, dtype=torch.bfloat16)
    with pytest.raises((ValueError, RuntimeError)):
        cache(x, x, torch.zeros(1, 2, 1, 16, dtype=torch.bfloat16))
    assert cache.lengths.tolist() == [0]


def test_accounting_counts_the_rows_in_use():
    from types import SimpleNamespace

    from logkv_amd import cache_compression_snapshot

    cache = EvictingKVCache(2, 4, 8, 8, 16, scale=1.0, device="cpu")
    cache.lengths.copy_(torch.tensor([16, 9], dtype=torch.int32))
    model = SimpleNamespace(transformer=SimpleNamespace(h=[SimpleNamespace(attn=SimpleNamespace(kv_cache=cache))]))
    counts = cache_compression_snapshot(model, 100)
    assert counts["retained_slots"] == 25 * 4 and counts["dense_slots"] == 100 * 8 and counts["layer_group_count"] == 8
