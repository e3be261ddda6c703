"""Inference streaming over a LogStructuredKVCache: block prefill and pending-token decode
pairing of CausalSelfAttention's LogKV path (litgpt/model.py:1125-1361, inference:
``defer_last_single=True``, no gradient).

The model's projections, RoPE and output projection are not on this path: the caller
hands over post-RoPE queries and keys, values and the pre-RoPE keys that routing uses,
and gets the attention output. Every attention runs in the HIP library
(``log_kv_chunk_attention``: pack + streaming / matrix-core kernels) and every commit
is the cache's ``add_recent`` (the flush kernels).
"""

from __future__ import annotations

import operator

import torch

from .log_kv_pack import log_kv_chunk_attention, log_kv_draft_attention


def _cols(rows, start, end):
    """Columns [start, end) of per-row span flags (host lists or a [B, T] tensor)."""
    if rows is None:
        return None
    if isinstance(rows, torch.Tensor):
        return rows[:, start:end]
    return [row[start:end] for row in rows]


def _join(a, b):
    """Span flags of a block followed by another (lists or tensors)."""
    if isinstance(a, torch.Tensor) or isinstance(b, torch.Tensor):
        dev = (a if isinstance(a, torch.Tensor) else b).device
        return torch.cat([torch.as_tensor(x, dtype=torch.uint8, device=dev) for x in (a, b)], dim=1)
    return [list(x) + list(y) for x, y in zip(a, b)]


def _join_pos(a, b):
    """Positions (``[n]`` or ``[B, n]``) of a block followed by another, None where either is."""
    if a is None or b is None:
        return None
    a = a.to(b.device)
    if a.dim() != b.dim():
        rows = (a if a.dim() == 2 else b).size(0)
        a, b = (x if x.dim() == 2 else x.expand(rows, -1) for x in (a, b))
    return torch.cat([a, b], dim=-1)


def _check_path(path, tokens, batch):
    """The accepted tokens as one list of indices per batch row (or one for all), each in the draft's order."""
    if hasattr(path, "tolist"):
        path = path.tolist() if path.ndim else [path.item()]
    path = list(path)
    if not path:
        return [[]]
    try:
        rows = [list(row) for row in path] if isinstance(path[0], (list, tuple)) else [path]
        rows = [[i.item() if hasattr(i, "item") else i for i in row] for row in rows]
        if any(isinstance(i, bool) for row in rows for i in row):
            raise TypeError("a mask")
        rows = [[operator.index(i) for i in row] for row in rows]
    except TypeError as e:
        raise ValueError("path must hold indices of drafted tokens") from e
    if len(rows) not in (1, batch) or len({len(row) for row in rows}) != 1:
        raise ValueError("path must be [n] or [B, n] indices of drafted tokens, as many in every batch row")
    for row in rows:
        if any(not 0 <= i < tokens for i in row) or any(i >= j for i, j in zip(row, row[1:])):
            raise ValueError("path must hold increasing indices of drafted tokens")
    return rows


def _pick(x, index):
    """Columns ``index [1 or B, n]`` (device) of per-token rows ``x [B, G, T, d]``."""
    if index.size(0) == 1:
        return x.index_select(2, index[0])
    return x.gather(2, index[:, None, :, None].expand(-1, x.size(1), -1, x.size(3)))


class LogKVStreamingAttention:
    """The streaming engine of one attention layer over ``cache``.

    ``__call__(q, k, v, k_raw, input_pos, span_ends)`` processes T new tokens
    (q ``[B, n_head, T, d]`` post-RoPE, k / v ``[B, n_groups, T, d]`` post-RoPE keys and
    values, k_raw the pre-RoPE keys, input_pos ``[T]`` or ``[B, T]``, span_ends per-row
    flags when the cache has an Alpha exact pool) and returns ``[B, T, n_head * dv]``:

    * a token left pending by the previous call is paired with the first new token: that
      token's query attends to the cache plus both (non-causal among the two), then both
      are committed (litgpt/model.py:1226-1250);
    * the rest runs in blocks of ``max(2, min(prefill_block, recent_size))`` tokens: the
      block's queries attend to the cache state at the block's start plus the block's own
      tokens causally, then the block is committed; a lone final token of odd length is
      attended but kept pending (litgpt/model.py:1252-1340), so prefill and decode keep
      the 2-token commit boundaries of the concatenated sequence.

    The pending tuple is ``_log_kv_pending`` (keys, values, pre-RoPE keys, positions,
    span flags), the attribute the compression accounting reads.

    Speculative decoding: ``draft`` attends a tree of drafted tokens without committing any,
    ``accept`` commits those of them that the model confirms. No counterpart in the reference.
    """

    def __init__(self, cache, scale: float, prefill_block: int = 2048):
        if not cache.semantic_clusters:
            raise NotImplementedError("streaming runs on the semantic LogKV cache")
        self.cache = cache
        self.scale = float(scale)
        self.prefill_block = int(prefill_block)
        self._log_kv_pending = None
        self._drafted = None      # the last draft's rows, until accept or the next call

    @property
    def kv_cache(self):
        return self.cache

    def reset(self) -> None:
        """Empty the cache and drop the pending token (a new request)."""
        self.cache.reset_parameters()
        self._log_kv_pending = None
        self._drafted = None

    def _check_tokens(self, tokens, span_ends):
        if tokens < 1:
            raise ValueError("at least one token per call")
        if self.cache.alpha_exact_tokens and span_ends is None:
            raise ValueError("an Alpha exact pool needs span boundary flags for every streamed token")

    @torch.no_grad()
    def __call__(self, q, k, v, k_raw, input_pos=None, span_ends=None):
        B, _, T, _ = q.shape
        self._check_tokens(T, span_ends)
        self._drafted = None
        outputs = self._advance(q, k, v, k_raw, input_pos, span_ends)
        y = outputs[0] if len(outputs) == 1 else torch.cat(outputs, dim=2)   # [B, n_head, T, dv]
        return y.transpose(1, 2).reshape(B, T, -1)

    @torch.no_grad()
    def draft(self, q, k, v, k_raw, visible, input_pos=None, span_ends=None):
        """Attention of T drafted tokens, ``[B, T, n_head * dv]``, over the cache, a token left pending and the drafted
        tokens that ``visible`` (bool, ``[T, T]`` or ``[B, T, T]``) shows each: a tree's mask has a token's ancestors
        and itself. The other arguments are those of a call, RoPE and ``input_pos`` at each token's depth; a token
        stands behind its ancestors. Nothing is committed: the tensors are held, not copied, for ``accept``, and
        dropped by the next draft, call or reset."""
        T = q.size(2)
        self._check_tokens(T, span_ends)
        if k_raw.shape[:3] != k.shape[:3] or (input_pos is not None and input_pos.size(-1) != T):
            raise ValueError("k_raw and input_pos must match the drafted tokens")
        pending = self._log_kv_pending
        y = log_kv_draft_attention(self.cache, q, k, v, visible, self.scale,
                                   pending=None if pending is None else pending[:2])
        self._drafted = (k, v, k_raw, input_pos, span_ends)
        return y.transpose(1, 2).reshape(q.size(0), T, -1)

    @torch.no_grad()
    def accept(self, path) -> None:
        """Commit the last draft's tokens ``path`` (increasing indices, ``[n]`` or ``[B, n]``, on the host; none drops
        the draft) as a call with those tokens would: a pending token pairs with the first, a lone last one is kept
        pending. The drafted outputs stand for the call's."""
        if self._drafted is None:
            raise RuntimeError("accept() needs a draft() that no other call followed")
        k, v, k_raw, pos, ends = self._drafted
        rows = _check_path(path, k.size(2), k.size(0))
        self._drafted = None
        n = len(rows[0])
        if not n:
            return
        if rows == [list(range(n))]:     # a chain's prefix
            k, v, k_raw = k[:, :, :n], v[:, :, :n], k_raw[:, :, :n]
            pos, ends = None if pos is None else pos[..., :n], _cols(ends, 0, n)
        else:
            host = torch.tensor(rows, dtype=torch.int64)
            index = host.pin_memory().to(k.device, non_blocking=True) if k.is_cuda else host
            k, v, k_raw = _pick(k, index), _pick(v, index), _pick(k_raw, index)
            if pos is not None:
                where = index.to(pos.device)
                pos = pos[where[0]] if pos.dim() == len(rows) == 1 else torch.gather(
                    pos.expand(k.size(0), -1), 1, where.expand(k.size(0), -1))
            if isinstance(ends, torch.Tensor):
                ends = ends.gather(1, index.to(ends.device).expand(k.size(0), -1))
            elif ends is not None:
                ends = [[row[i] for i in rows[b % len(rows)]] for b, row in enumerate(ends)]
        self._advance(None, k, v, k_raw, pos, ends)

    def _advance(self, q, k, v, k_raw, input_pos, span_ends):
        """Commits the tokens, attending before each commit where queries are given; returns the outputs."""
        cache, T = self.cache, k.size(2)

        def pos_slice(a, b):
            if input_pos is None:
                return None
            return input_pos[a:b] if input_pos.dim() == 1 else input_pos[:, a:b]

        outputs, start = [], 0
        pending = self._log_kv_pending
        if pending is not None:
            pk, pv, pk_raw, ppos, pends = pending
            # The pair's keys and values serve the attention and the commit.
            kk, vv = torch.cat([pk, k[:, :, :1]], dim=2), torch.cat([pv, v[:, :, :1]], dim=2)
            if q is not None:
                outputs.append(log_kv_chunk_attention(cache, q[:, :, :1], kk, vv, self.scale, 0.0, causal_tail=0,
                                                      reuse_prefix=True))
            pos = _join_pos(ppos, pos_slice(0, 1))
            ends = None if pends is None else _join(pends, _cols(span_ends, 0, 1))
            cache.add_recent(kk, vv, k_raw=torch.cat([pk_raw, k_raw[:, :, :1]], dim=2), input_pos=pos,
                             span_ends=ends)
            self._log_kv_pending = None
            start = 1

        blk_size = max(2, min(self.prefill_block, cache.recent_size))
        while start < T:
            end = min(T, start + blk_size)
            defer_tail = end == T and (end - start) % 2 == 1
            commit_end = end - 1 if defer_tail else end
            if q is not None:
                outputs.append(log_kv_chunk_attention(cache, q[:, :, start:end], k[:, :, start:end],
                                                      v[:, :, start:end], self.scale, 0.0, reuse_prefix=True))
            if commit_end > start:
                cache.add_recent(k[:, :, start:commit_end], v[:, :, start:commit_end],
                                 k_raw=k_raw[:, :, start:commit_end], input_pos=pos_slice(start, commit_end),
                                 span_ends=_cols(span_ends, start, commit_end))
            if defer_tail:
                self._log_kv_pending = (k[:, :, commit_end:end], v[:, :, commit_end:end],
                                        k_raw[:, :, commit_end:end], pos_slice(commit_end, end),
                                        _cols(span_ends, commit_end, end))
            start = end
        return outputs
