"""An exact K/V cache of a fixed budget: rows are kept by the attention weight that they have drawn.

The uncompressed counterpart of a ``LogStructuredKVCache`` for layers or requests that keep exact rows. No
counterpart in the reference, whose dense cache grows with the sequence.
"""

from __future__ import annotations

import math

import torch

from ._lib import check_activation_dtype
from .row_attention import (_ROW_DTYPES, EvictedRows, _workspace_bytes, log_kv_evict, log_kv_tree_attention,
                            log_kv_weight_attention)


class EvictingKVCache:
    """Rows ``[batch, n_groups, budget + block, d]`` of which at most ``budget`` outlive an eviction.

    ``cache(q, k, v, counts=None)`` attends T new tokens causally over the rows and each other, adds every row's
    probabilities to its weight and appends the new rows; when they do not fit, every (batch row, KV head) is first cut
    to its last ``recent`` rows and, up to ``budget`` in all, its others of largest weight. ``cache.draft(q, k, v,
    visible)`` attends a tree of drafted tokens without a change: commit the accepted ones with a call.

    Calls longer than ``block`` tokens run in blocks (an eviction may fall between them); a refused call leaves the
    cache as it was. ``lengths`` (int32 ``[batch]``, on the device) are the rows in use; the host keeps only an upper
    bound of them and never waits. Eviction copies into a second set of buffers, which swaps with the first. Keys are
    kept as given, post-RoPE at the tokens' own positions; with ``track_positions`` the ordinal of each row's token
    stands in ``positions`` (int64 ``[batch, n_groups, capacity]``). Its calls cannot be captured into a HIP graph: the
    host's bound decides when to evict, and eviction swaps the buffers."""

    def __init__(self, batch_size: int, n_groups: int, k_dim: int, v_dim: int, budget: int, *, scale: float,
                 recent: int | None = None, block: int | None = None, dtype=torch.bfloat16, device="cuda",
                 track_positions: bool = False) -> None:
        recent = budget // 4 if recent is None else recent
        block = max(1, budget // 4) if block is None else block
        if min(batch_size, n_groups, k_dim, v_dim, budget, block) < 1 or not 0 <= recent <= budget:
            raise ValueError("sizes, budget and block must be positive, recent between 0 and the budget")
        if dtype not in _ROW_DTYPES:
            raise ValueError("the cache must be bfloat16 or float16")
        if not 0.0 < scale < math.inf:
            raise ValueError("attention scale must be positive")
        _workspace_bytes(True, batch_size, n_groups, n_groups, 1, budget + block, k_dim, v_dim, _ROW_DTYPES[dtype])
        self.batch_size, self.n_groups, self.budget, self.recent, self.block = batch_size, n_groups, budget, recent, block
        self.scale, self.capacity = float(scale), budget + block
        shape = (batch_size, n_groups, self.capacity)

        def buffers():
            return EvictedRows(
                torch.zeros(*shape, k_dim, dtype=dtype, device=device),
                torch.zeros(*shape, v_dim, dtype=dtype, device=device),
                torch.zeros(shape, dtype=torch.float32, device=device),
                torch.full(shape, -1, dtype=torch.int64, device=device) if track_positions else None,
                torch.full((*shape[:2], budget), -1, dtype=torch.int32, device=device),
                torch.zeros(batch_size, dtype=torch.int32, device=device))

        self._rows, self._spare = buffers(), buffers()
        self._tokens = torch.zeros(batch_size, dtype=torch.int64, device=device) if track_positions else None
        self._bound = 0          # no batch row has more rows than this

    @property
    def k(self):
        return self._rows.k

    @property
    def v(self):
        return self._rows.v

    @property
    def weights(self):
        return self._rows.weights

    @property
    def positions(self):
        return self._rows.positions

    @property
    def lengths(self):
        return self._rows.lengths

    def reset(self) -> None:
        """Empty the cache (a new request)."""
        self._rows.lengths.zero_()
        if self._tokens is not None:
            self._tokens.zero_()
        self._bound = 0

    @torch.no_grad()
    def evict(self) -> torch.Tensor:
        """Cut every lane to the budget now; returns the kept rows' indices before (int32 ``[batch, n_groups,
        budget]``, -1 behind the last), valid until the next eviction but one."""
        self._refuse_capture()
        old = self._rows
        self._rows = log_kv_evict(old.k, old.v, old.weights, old.lengths, self.budget, recent=self.recent,
                                  positions=old.positions, out=self._spare)
        self._spare = old
        self._bound = min(self._bound, self.budget)
        return self._rows.kept

    @torch.no_grad()
    def draft(self, q, k, v, visible):
        """Attention of drafted tokens ``[batch, n_heads, T, v_dim]`` over the rows and the drafted rows visible to
        each (``log_kv_tree_attention``); the cache stays as it is."""
        self._refuse_capture()
        return log_kv_tree_attention(q, k, v, self.k, self.v, self.lengths, visible, self.scale)

    @torch.no_grad()
    def __call__(self, q, k, v, counts=None):
        """Attention ``[batch, n_heads, T, v_dim]`` of T new tokens, which join the cache. ``counts`` (int32
        ``[batch]`` on the device) gives the tokens that exist per row of a padded batch."""
        self._refuse_capture()
        tokens = self._check_call(q, k, v, counts)
        outputs = []
        for start in range(0, tokens, self.block):
            end = min(tokens, start + self.block)
            part = None if counts is None else (counts - start).clamp(0, end - start).to(torch.int32)
            outputs.append(self._step(q[:, :, start:end], k[:, :, start:end], v[:, :, start:end], part))
        return outputs[0] if len(outputs) == 1 else torch.cat(outputs, dim=2)

    def _check_call(self, q, k, v, counts):
        """The call's tokens; refuses what any of its blocks would, before a row is dropped or stored."""
        batch, groups, dk, dv, device = self.batch_size, self.n_groups, self.k.size(3), self.v.size(3), self.k.device
        heads, tokens = q.shape[1:3] if q.ndim == 4 else (0, 0)
        if (tokens < 1 or q.shape != (batch, heads, tokens, dk) or heads < 1 or heads % groups
                or k.shape != (batch, groups, tokens, dk) or v.shape != (batch, groups, tokens, dv)
                or not q.device == k.device == v.device == device
                or counts is not None and (counts.shape != (batch,) or counts.dtype not in (torch.int32, torch.int64)
                                           or counts.device != device)):
            raise ValueError("a call takes at least one token: q [B, n_heads, T, d], k and v [B, G, T, d], counts [B], "
                             "all on the cache's device")
        for x in (q, k, v):
            check_activation_dtype(x.dtype)
        # The sizes that an attention refuses.
        _workspace_bytes(True, batch, heads, groups, min(tokens, self.block), self.capacity, dk, dv, _ROW_DTYPES[self.k.dtype])
        return tokens

    def _step(self, q, k, v, counts):
        n = q.size(2)
        if self._bound + n > self.capacity:
            self.evict()
        rows = self._rows
        out = log_kv_weight_attention(q, k, v, rows.k, rows.v, rows.weights, rows.lengths, self.scale, counts=counts)
        if self._tokens is not None:
            # Columns of tokens that do not exist lie behind the row's last and are written over later.
            step = torch.arange(n, device=q.device)
            at = rows.lengths[:, None] + step
            rows.positions.scatter_(2, at[:, None].expand(-1, self.n_groups, -1).long(),
                                    (self._tokens[:, None] + step)[:, None].expand(-1, self.n_groups, -1))
            self._tokens += n if counts is None else counts
        rows.lengths.add_(n if counts is None else counts)
        self._bound += n
        return out

    def _refuse_capture(self):
        if self.k.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("an EvictingKVCache's calls cannot be captured: capture log_kv_weight_attention on its "
                               "rows instead")
