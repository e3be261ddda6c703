"""Attention over an exact cache's rows and the rows of the call itself, and eviction by attention weight.

Rows are ``[batch, groups, capacity, features]`` (bfloat16 or float16), ``lengths`` the rows in use per
batch row. No counterpart in the reference, whose LogKV path masks nothing among its in-flight rows but
the causal tail and keeps no exact cache that attention weight cuts:

* ``log_kv_tree_attention``: a tree of drafted tokens over a cache that is only read, for the
  verification step of speculative decoding (``LogKVStreamingAttention.draft`` runs it over the
  compressed cache's packed rows, with their log-mass as bias);
* ``log_kv_weight_attention``: causal attention of new tokens that adds each row's probability to its
  running weight and stores the new rows behind the cache's;
* ``log_kv_evict``: the rows of every (batch row, KV head) cut to a budget by those weights
  (``EvictingKVCache`` runs the three of them over its own rows).

All run in liblogkv_hip.so on the current stream of the tensors' device, allocate their outputs and
scratch through torch, never wait for the host and can be captured into a HIP graph. They are for
inference: none has a gradient.
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import NamedTuple

import torch

from ._lib import check, check_activation_dtype, require_device
from ._rows import BF16, F16, RowsArgs, pack_evict, pack_rows, rows_lib

_ROW_DTYPES = {torch.bfloat16: BF16, torch.float16: F16}
_LENGTH_DTYPES = (torch.int32, torch.int64)
_NO_STRIDES = (0, 0, 0)


class EvictedRows(NamedTuple):
    """What ``log_kv_evict`` keeps: rows ``k / v [B, G, keep, d]``, ``weights`` and ``positions [B, G, keep]``,
    ``kept`` (int32 ``[B, G, keep]``, the rows' indices before, -1 behind the last) and ``lengths`` (int32 ``[B]``)."""

    k: torch.Tensor
    v: torch.Tensor
    weights: torch.Tensor
    positions: torch.Tensor | None
    kept: torch.Tensor
    lengths: torch.Tensor


def _launch(entry, what, index, *args):
    """Calls a C entry point on the current stream of the device ``index``, made the current one."""
    if torch._C._cuda_getDevice() == index:
        return check(entry(*args, torch._C._cuda_getCurrentRawStream(index)), what)
    with torch.cuda.device(index):
        return check(entry(*args, torch._C._cuda_getCurrentRawStream(index)), what)


def _no_gradient():
    return NotImplementedError("row attention is for inference: it has no gradient (run it under torch.no_grad())")


def _small_rows(x, dtype):
    """Rows of the call in the cache's dtype, readable in 16-byte units."""
    if x.dtype != dtype:
        check_activation_dtype(x.dtype)
        x = x.to(dtype)
    sb, sh, st, sd = x.stride()
    if sd != 1 or (sb | sh | st) & 7 or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)   # of any strides, also those of size-1 dimensions
    return x


def _row_strides(x):
    """Strides of the first three dimensions, 0 for those of one element (theirs are never taken)."""
    return tuple(0 if n == 1 else s for n, s in zip(x.shape[:3], x.stride()))


def _contiguous_rows(x):
    return x.stride(2) == 1 or x.size(2) == 1


def _lengths(lengths, batch, cap, index, room=0):
    """(int32 tensor or None, its address, its stride, added rows) of an int or an int tensor ``[B]``."""
    if isinstance(lengths, torch.Tensor):
        if lengths.shape != (batch,) or lengths.get_device() != index or lengths.dtype not in _LENGTH_DTYPES:
            raise ValueError("lengths must be an int or an int32 tensor [batch] on the cache's device")
        if lengths.dtype != torch.int32 or not lengths.is_contiguous():
            lengths = lengths.to(torch.int32).contiguous()
        return lengths, lengths.data_ptr(), 1, 0
    lengths = int(lengths)
    if not 0 <= lengths <= cap - room:
        raise ValueError(f"{lengths} rows and {room} new ones do not fit the cache's {cap}")
    return None, 0, 0, lengths


@lru_cache(maxsize=256)
def _workspace_bytes(weights, batch, heads, groups, tq, cap, dk, dv, dtype):
    """Scratch of a call of these sizes."""
    args = RowsArgs(n_batch=batch, n_heads=heads, n_groups=groups, tq=tq, cap=cap, dk=dk, dv=dv, dtype=dtype,
                    weights=1 if weights else 0)
    need = rows_lib().logkv_rows_workspace_bytes(bytes(args))
    if need < 0:
        raise ValueError("row attention: " + rows_lib().logkv_last_error().decode(errors="replace"))
    return need


def _attention(q, k, v, cache_k, cache_v, scale, lengths, room, *, bias=None, visible=None, counts=None, weights=None,
               in_use=None, bias_scale=1.0):
    """Checks and launch of both attentions. ``in_use`` in place of ``lengths``: (address, stride) of device counts
    per batch row, a second count's address (0: none) and rows to add to both. ``bias_scale``: a factor of the bias."""
    if not q.ndim == k.ndim == v.ndim == cache_k.ndim == cache_v.ndim == 4:
        raise ValueError("queries, rows and cache must be 4-dimensional")
    batch, heads, tq, dk = q.shape
    k_shape, v_shape = cache_k.shape, cache_v.shape
    groups, cap, dv = k_shape[1], k_shape[2], v_shape[3]
    dtype, index = cache_k.dtype, cache_k.get_device()
    code = _ROW_DTYPES.get(dtype)
    if code is None or cache_v.dtype != dtype:
        raise ValueError("the cache must be bfloat16 or float16")
    if (k_shape != (batch, groups, cap, dk) or v_shape != (batch, groups, cap, dv) or groups < 1
            or heads % groups or heads < 1 or tq < 1 or batch < 1):
        raise ValueError("cache rows must be [B, G, capacity, d] with G dividing the query heads")
    if k.shape != (batch, groups, tq, dk) or v.shape != (batch, groups, tq, dv):
        raise ValueError("the call's rows must be [B, G, T, d], one per query position")
    require_device(cache_k, "cache_k")
    if not cache_v.get_device() == q.get_device() == k.get_device() == v.get_device() == index:
        raise ValueError("all tensors must be on the cache's device")
    if not (0.0 < scale < math.inf):
        raise ValueError("attention scale must be positive")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or cache_k.requires_grad
                                    or cache_v.requires_grad or bias is not None and bias.requires_grad):
        raise _no_gradient()
    ck, cv = cache_k.data_ptr(), cache_v.data_ptr()
    ck_sb, ck_sg, ck_st, ck_sd = cache_k.stride()
    cv_sb, cv_sg, cv_st, cv_sd = cache_v.stride()
    if cap and (ck_sd != 1 or cv_sd != 1 or (ck_sb | ck_sg | ck_st | cv_sb | cv_sg | cv_st) & 7 or (ck | cv) & 15):
        ck_sb, ck_sg, ck_st = _row_strides(cache_k)
        cv_sb, cv_sg, cv_st = _row_strides(cache_v)
        if ck_sd != 1 or cv_sd != 1 or (ck_sb | ck_sg | ck_st | cv_sb | cv_sg | cv_st) & 7 or (ck | cv) & 15:
            raise ValueError("cache rows must be 16-byte aligned with contiguous features")
    out_dtype = q.dtype
    q_st, k_st, v_st = q.stride(), k.stride(), v.stride()
    qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (q.dtype != dtype or k.dtype != dtype or v.dtype != dtype or not q_st[3] == k_st[3] == v_st[3] == 1
            or (q_st[0] | q_st[1] | q_st[2] | k_st[0] | k_st[1] | k_st[2] | v_st[0] | v_st[1] | v_st[2]) & 7
            or (qp | kp | vp) & 15):
        q, k, v = _small_rows(q, dtype), _small_rows(k, dtype), _small_rows(v, dtype)
        q_st, k_st, v_st = q.stride(), k.stride(), v.stride()
        qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    n2_ptr = 0
    if in_use is None:
        lengths, n_ptr, n_st, len_add = _lengths(lengths, batch, cap, index, room)
    else:
        n_ptr, n_st, n2_ptr, len_add = in_use
    b_ptr, b_st, b_half = 0, _NO_STRIDES, 0
    if bias is not None:
        if bias.shape != (batch, groups, cap) or bias.get_device() != index or bias.dtype not in (torch.float32, dtype):
            raise ValueError("bias must be [B, G, capacity] on the cache's device, float32 or the cache's dtype")
        b_ptr, b_st, b_half = bias.data_ptr(), bias.stride(), int(bias.dtype == dtype)
    vis_ptr = vis_sb = vis_st = w_ptr = w_sb = w_sg = 0
    if visible is not None:
        vis_ptr, vis_sb, vis_st = visible.data_ptr(), visible.stride(0) if visible.ndim == 3 else 0, visible.stride(-2)
    else:
        w_ptr, (w_sb, w_sg, _) = weights.data_ptr(), weights.stride()
    out = cache_k.new_empty((batch, heads, tq, dv))
    need = _workspace_bytes(weights is not None, batch, heads, groups, tq, cap, dk, dv, code)
    workspace = cache_k.new_empty(need // 2)
    o_sh = tq * dv
    args = pack_rows(
        qp, *q_st[:3], kp, *k_st[:3], vp, *v_st[:3], ck, ck_sb, ck_sg, ck_st, cv, cv_sb, cv_sg, cv_st,
        b_ptr, *b_st, n_ptr, n2_ptr, vis_ptr, vis_sb, vis_st,
        0 if counts is None else counts.data_ptr(), w_ptr, w_sb, w_sg, out.data_ptr(), heads * o_sh, o_sh, dv,
        batch, heads, groups, tq, cap, dk, dv, code, n_st, len_add, b_half, scale, bias_scale)
    handle = rows_lib()
    if weights is None:
        _launch(handle.logkv_tree_attention, "logkv_tree_attention", index, args, workspace.data_ptr(), need)
    else:
        _launch(handle.logkv_weight_attention, "logkv_weight_attention", index, args, workspace.data_ptr(), need)
    return out if out_dtype == dtype else out.to(out_dtype)


def log_kv_tree_attention(q, k, v, cache_k, cache_v, lengths, visible, scale, *, bias=None):
    """Attention of T drafted tokens over a cache and each other, ``[B, n_heads, T, dv]``.

    ``q [B, n_heads, T, dk]``, the drafted rows ``k [B, G, T, dk]`` and ``v [B, G, T, dv]``; ``cache_k / cache_v
    [B, G, capacity, d]`` with ``lengths`` rows in use (an int, or an int32 tensor ``[B]`` read on the device and
    held to the capacity). Every token sees all rows in use, and the drafted row r where ``visible[t, r]`` (bool,
    ``[T, T]`` or ``[B, T, T]``; a tree's mask has each token's ancestors and itself). ``bias`` (``[B, G, capacity]``,
    float32 or the cache's dtype, any strides) is added to the scaled logits; -inf hides a row. A token that sees
    nothing gets zeros, and what hidden rows hold (NaN, infinities) reaches no output.

    Queries and drafted rows of another activation dtype are rounded to the cache's, and the output is returned
    in the queries'. The cache is only read: commit the accepted tokens with the cache's own call."""
    return _attention(q, k, v, cache_k, cache_v, float(scale), lengths, 0, bias=bias,
                      visible=_tree(visible, q, cache_k))


def _tree(visible, q, cache_k):
    """The checked mask of a draft, with contiguous rows."""
    if not isinstance(visible, torch.Tensor) or q.ndim != 4:
        raise ValueError("visible must be a bool tensor [T, T] or [B, T, T], queries [B, n_heads, T, d]")
    tokens, shape = q.size(2), visible.shape
    if (visible.dtype not in (torch.bool, torch.uint8)
            or not (shape == (tokens, tokens) or shape == (q.size(0), tokens, tokens))
            or visible.get_device() != cache_k.get_device()):
        raise ValueError("visible must be a bool tensor [T, T] or [B, T, T] on the cache's device")
    return visible if visible.stride(-1) == 1 else visible.contiguous()


def log_kv_weight_attention(q, k, v, cache_k, cache_v, weights, lengths, scale, *, counts=None):
    """Causal attention of T new tokens over a cache and themselves, ``[B, n_heads, T, dv]``, that keeps the
    rows' attention weights.

    In place, with n = ``lengths[b]`` rows in use: ``weights[b, g, j] += sum of row j's probabilities`` over the KV
    head's query heads and the T queries for j < n, ``weights[b, g, n + t]`` set to new row t's sum, and the new rows
    stored at cache rows n + t. ``lengths`` itself is left to the caller (the rows in use are n + T afterwards); as
    an int tensor it is read on the device, and rows past the capacity are attended to but not stored. ``counts``
    (int32 ``[B]``) gives the tokens that really exist per batch row of a padded batch: the others' outputs are zeros,
    they add no weight and are not stored. ``weights`` is float32 ``[B, G, capacity]`` with contiguous rows."""
    batch, _, cap = shape = cache_k.shape[:3]
    if (weights.shape != shape or weights.dtype != torch.float32 or weights.get_device() != cache_k.get_device()
            or not _contiguous_rows(weights) or cap < 1):
        raise ValueError("weights must be float32 [B, G, capacity] on the cache's device with contiguous rows")
    if _repeats(weights) or _repeats(cache_k) or _repeats(cache_v):
        raise ValueError("weights and cache are written: their rows must not share memory (expanded tensors)")
    if weights.requires_grad and torch.is_grad_enabled():
        raise _no_gradient()
    if counts is not None:
        if (counts.shape != (batch,) or counts.get_device() != cache_k.get_device()
                or counts.dtype not in _LENGTH_DTYPES):
            raise ValueError("counts must be an int32 tensor [batch] on the cache's device")
        counts = counts.to(torch.int32).contiguous()
    return _attention(q, k, v, cache_k, cache_v, float(scale), lengths, q.size(2), counts=counts, weights=weights)


def _repeats(t):
    """Whether elements of an expanded tensor share memory."""
    return 0 in t.stride() and any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape))


def _span(t):
    """First and one past the last byte that a tensor's elements occupy."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + last * t.element_size()


def _unit_strides(t):
    """Strides of rows that are read in 16-byte units, None where they cannot be."""
    sb, sg, st, sd = t.stride()
    size, at = t.element_size(), t.data_ptr()
    if ((sb | sg | st) * size | at) & 15:
        sb, sg, st = _row_strides(t)
    return (sb, sg, st) if sd == 1 and not ((sb | sg | st) * size | at) & 15 else None


def log_kv_evict(cache_k, cache_v, weights, lengths, keep, *, recent=0, positions=None, out=None):
    """Cut every (batch row, KV head) of a cache to its last ``recent`` rows and, up to ``keep`` in all, its other
    rows of largest weight, kept in their order; returns ``EvictedRows``.

    ``cache_k / cache_v [B, G, capacity, d]`` (rows of a multiple of 16 bytes, of 1, 2 or 4 byte elements), ``weights``
    float32 ``[B, G, capacity]``, ``lengths`` an int or an int32 tensor ``[B]``, ``positions`` optionally int64
    ``[B, G, capacity]``. Equal weights keep the lowest index, NaN counts as the largest. A sequence of at most
    ``keep`` rows keeps them all; rows behind a sequence's last are zeros (-1 in ``kept`` and ``positions``).

    The result is new tensors, or ``out``: an ``EvictedRows`` of buffers of at least ``keep`` rows that do not overlap
    the inputs (a cache's second buffer set), of which the first ``keep`` rows are written."""
    if cache_k.ndim != 4 or cache_v.ndim != 4 or cache_k.shape[:3] != cache_v.shape[:3]:
        raise ValueError("cache rows must be [B, G, capacity, d]")
    batch, groups, cap, dk = cache_k.shape
    dv, dtype, index = cache_v.size(3), cache_k.dtype, cache_k.get_device()
    keep, recent = int(keep), int(recent)
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError("keep must be at least 1, recent between 0 and keep")
    require_device(cache_k, "cache_k")
    if cache_v.dtype != dtype or not cache_v.get_device() == weights.get_device() == index:
        raise ValueError("all tensors must be on the cache's device, keys and values of one dtype")
    if weights.shape != (batch, groups, cap) or weights.dtype != torch.float32 or not _contiguous_rows(weights):
        raise ValueError("weights must be float32 [B, G, capacity] with contiguous rows")
    p_in = p_out = _NO_STRIDES
    if positions is not None:
        p_in = (positions.data_ptr(), *positions.stride()[:2])
        if (positions.shape != (batch, groups, cap) or positions.dtype != torch.int64 or not _contiguous_rows(positions)
                or positions.get_device() != index):
            raise ValueError("positions must be int64 [B, G, capacity] with contiguous rows")
    ck_st, cv_st = _unit_strides(cache_k), _unit_strides(cache_v)
    if ck_st is None or cv_st is None:
        raise ValueError("cache rows must be 16-byte aligned with contiguous features")
    if torch.is_grad_enabled() and (cache_k.requires_grad or cache_v.requires_grad or weights.requires_grad):
        raise _no_gradient()
    lengths, n_ptr, _, len_add = _lengths(lengths, batch, cap, index)
    if out is None:
        kept = weights.new_empty((batch, groups, keep), dtype=torch.int32)
        out = EvictedRows(
            cache_k.new_empty((batch, groups, keep, dk)), cache_v.new_empty((batch, groups, keep, dv)),
            weights.new_empty((batch, groups, keep)),
            None if positions is None else positions.new_empty((batch, groups, keep)), kept, kept.new_empty(batch))
        k, v, w, p, kept, n = out
        k_st, v_st = k.stride()[:3], v.stride()[:3]
    else:
        _check_evict_out(out, cache_k, cache_v, weights, positions, lengths, keep)
        k, v, w, p, kept, n = out
        k_st, v_st = _unit_strides(k), _unit_strides(v)
    if p is not None:
        p_out = (p.data_ptr(), *p.stride()[:2])
    args = pack_evict(
        cache_k.data_ptr(), *ck_st, cache_v.data_ptr(), *cv_st, weights.data_ptr(),
        *weights.stride()[:2], *p_in, n_ptr, k.data_ptr(), *k_st, v.data_ptr(), *v_st, w.data_ptr(),
        *w.stride()[:2], *p_out, kept.data_ptr(), n.data_ptr(), batch, groups, cap, dk, dv, cache_k.element_size(),
        len_add, keep, recent)
    _launch(rows_lib().logkv_evict_rows, "logkv_evict_rows", index, args)
    return out


def _check_evict_out(out, cache_k, cache_v, weights, positions, lengths, keep):
    batch, groups, _, dk = cache_k.shape
    dv, device = cache_v.size(3), cache_k.device
    k, v, w, p, kept, n = out

    def rows(t, dtype, *rest):
        return (t.ndim == 3 + len(rest) and t.shape[:2] == (batch, groups) and t.size(2) >= keep and t.shape[3:] == rest
                and t.dtype == dtype and t.device == device and (t.stride(3) == 1 if rest else _contiguous_rows(t)))

    if not (rows(k, cache_k.dtype, dk) and rows(v, cache_k.dtype, dv) and rows(w, torch.float32)
            and _unit_strides(k) and _unit_strides(v) and (p is None) == (positions is None)
            and (p is None or rows(p, torch.int64)) and kept.shape == (batch, groups, keep) and kept.is_contiguous()
            and kept.dtype == torch.int32 and kept.device == device and n.shape == (batch,) and n.is_contiguous()
            and n.dtype == torch.int32 and n.device == device and not any(_repeats(t) for t in (k, v, w))
            and (p is None or not _repeats(p))):
        raise ValueError("out must be EvictedRows buffers of at least keep rows that match the cache")
    given = [t for t in (cache_k, cache_v, weights, positions, lengths) if t is not None]
    results = [t for t in out if t is not None]
    for i, t in enumerate(results):
        a, b = _span(t)
        for other in given + results[:i]:
            c, d = _span(other)
            if a < d and c < b:
                raise ValueError("out must not overlap the inputs or itself")
