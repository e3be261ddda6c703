"""An exact cache in pages: appends with the position rotation on the way, and attention of a batch whose sequences
share prefixes.

``k_pages / v_pages`` are ``[pages, groups, page_size, features]`` (bfloat16 or float16; page_size a power of two from
16 on), ``table`` int32 ``[batch, n]`` the pages of each sequence: its row i is slot ``i % page_size`` of page ``table[b, i
// page_size]``. No counterpart in the reference, whose caches are dense:

* ``log_kv_paged_append`` stores new tokens behind a sequence's rows, keys (and the queries beside them) rotated;
* ``log_kv_paged_attention`` attends new tokens over a prefix that several sequences share (a ``SharedPrefix``: pages,
  or rows of a cache, such as a compressed one's packed slots with their log-mass), their own rows and each other. A
  prefix's rows are read once for all of its sequences.

``PagedKVCache`` runs both over pages that it hands out. All run in liblogkv_hip.so on the current stream of the
tensors' device, allocate their outputs and scratch through torch, never wait for the host and can be captured into a
HIP graph. They are for inference: none has a gradient.
"""

from __future__ import annotations

import math
import operator
from functools import lru_cache
from typing import NamedTuple

import torch

from ._lib import check_activation_dtype, refuse_tangents, require_device
from ._paged import PagedArgs, pack_paged, pack_rotary, paged_lib
from .rotary import MAX_WIDTH, _NO_ROWS, _TYPES, _check_frequencies, _check_positions, _in_and_out
from .row_attention import (_LENGTH_DTYPES, _NO_STRIDES, _ROW_DTYPES, _int32, _launch, _lengths, _repeats, _small_rows, _tree,
                            _unit_strides)

MIN_PAGE = 16


class SharedPrefix(NamedTuple):
    """Prefixes of a batch: prefix i belongs to the i-th of as many equal runs of consecutive sequences.

    ``lengths`` (an int, or int32 ``[N]`` on the device) are the rows in use of each; the rows are those of pages of the
    sequences' own pool (``table`` int32 ``[N, n]``), or ``k / v [N, G, capacity, d]`` in the pages' dtype with an
    optional ``bias [N, G, capacity]`` (float32 or that dtype) that is added, times ``bias_scale``, to the scaled
    logits; -inf hides a row."""

    lengths: object
    table: torch.Tensor | None = None
    k: torch.Tensor | None = None
    v: torch.Tensor | None = None
    bias: torch.Tensor | None = None
    bias_scale: float = 1.0


def _check_pages(k_pages, v_pages, groups):
    """(dtype code, pages, page size, key and value widths) of a pool; its device is checked too."""
    shape, of_v, dtype = k_pages.shape, v_pages.shape, k_pages.dtype
    if len(shape) != 4 or len(of_v) != 4 or shape[0] != of_v[0] or not shape[1] == of_v[1] == groups or shape[2] != of_v[2]:
        raise ValueError("pages must be [pages, groups, page_size, d], keys and values alike")
    page = shape[2]
    if page < MIN_PAGE or page & (page - 1):
        raise ValueError(f"page_size must be a power of two from {MIN_PAGE} on, got {page}")
    code = _ROW_DTYPES.get(dtype)
    if code is None or v_pages.dtype != dtype:
        raise ValueError("the pages must be bfloat16 or float16")
    if not k_pages.is_cuda:
        require_device(k_pages, "k_pages")
    return code, shape[0], page, shape[3], of_v[3]


def _check_table(table, rows, index):
    shape, strides = table.shape, table.stride()
    if (len(shape) != 2 or shape[0] != rows or table.dtype is not torch.int32 or table.get_device() != index
            or shape[1] > 1 and strides[1] != 1):
        raise ValueError(f"a page table must be int32 [{rows}, n] on the pages' device with contiguous rows")
    return table.data_ptr(), strides[0], shape[1]


def _check_counts(counts, batch, index):
    if counts.shape != (batch,) or counts.get_device() != index or counts.dtype not in _LENGTH_DTYPES:
        raise ValueError("counts must be an int32 tensor [batch] on the pages' device")
    return _int32(counts)


def log_kv_paged_append(k, v, k_pages, v_pages, table, lengths, *, q=None, frequencies=None, positions=None, first=0,
                        interleaved=False, amplitude=1.0, counts=None):
    """Store T new tokens behind each sequence's rows and return (queries, keys) as rotated.

    ``k [B, G, T, dk]`` and ``v [B, G, T, dv]`` (bfloat16, float16 or float32, any strides) become rows ``lengths[b] + t``
    (an int, or an int32 tensor ``[B]``; left to the caller to advance), rounded to the pages' dtype once; with
    ``frequencies`` the keys, and ``q [B, n_heads, T, dk]`` where given, are rotated on the way as by ``log_kv_rotary``.
    A token's position is ``first`` (an int, or int64 ``[B]``: the position of a sequence's row 0) plus its row, or
    ``positions`` (int64 or int32 ``[T]`` or ``[B, T]``). ``counts`` (int32 ``[B]``) gives the tokens that exist per
    sequence of a padded batch; the others are rotated but not stored. Nor is a row whose page the table does not hold
    (an entry outside the pool, as -1, or behind its last).

    Returned are the rotated queries in their dtype (None without ``q``) and the keys in the pages' dtype, as
    ``log_kv_paged_attention`` takes them beside the rows before the call. Sequences must not share the pages that a
    call writes."""
    refuse_tangents(k, v, k_pages, v_pages, q, frequencies)
    k_shape, v_shape, dtype, index = k.shape, v.shape, k.dtype, k_pages.get_device()
    if len(k_shape) != 4 or len(v_shape) != 4 or v_shape[:3] != k_shape[:3] or k_shape[1] < 1:
        raise ValueError("new rows must be k [B, G, T, dk] and v [B, G, T, dv] of at least one group")
    batch, groups, tokens, dk = k_shape
    dv = v_shape[3]
    code, n_pages, page, k_width, v_width = _check_pages(k_pages, v_pages, groups)
    if v.dtype != dtype or not k.get_device() == v.get_device() == v_pages.get_device() == index:
        raise ValueError("new rows must be of one dtype, on the pages' device")
    if q is not None:
        q_shape = q.shape
        if (len(q_shape) != 4 or q_shape[0] != batch or q_shape[2] != tokens or q_shape[3] != dk or q.dtype != dtype
                or q.get_device() != index):
            raise ValueError("queries must be [B, n_heads, T, dk], in the new rows' dtype on their device")
    check_activation_dtype(dtype)
    kp_strides, vp_strides = k_pages.stride(), v_pages.stride()
    kp_sp, kp_sg, kp_st, kp_sd = kp_strides
    vp_sp, vp_sg, vp_st, vp_sd = vp_strides
    if k_width != dk or v_width != dv or not 1 <= dk <= MAX_WIDTH or not 1 <= dv <= MAX_WIDTH:
        raise ValueError(f"the pages' rows must be as wide as the new ones, up to {MAX_WIDTH} features")
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad
                                    or q is not None and q.requires_grad):
        raise NotImplementedError("a paged append is for inference: it has no gradient (run it under torch.no_grad())")
    if kp_sd != 1 and dk > 1 or vp_sd != 1 and dv > 1:
        raise ValueError("the pages' features must be contiguous")
    if 0 in kp_strides and _repeats(k_pages) or 0 in vp_strides and _repeats(v_pages):
        raise ValueError("pages are written: their rows must not share memory (expanded tensors)")
    amplitude = float(amplitude)
    if not math.isfinite(amplitude):
        raise ValueError("amplitude must be finite")
    table_ptr, table_sb, table_len = _check_table(table, batch, index)
    if table_len * page > 2 ** 30:
        raise ValueError("a sequence has at most 2^30 rows")
    lengths, n_ptr, _, len_add = _lengths(lengths, batch, table_len * page, index, tokens if counts is None else 0)
    c_ptr = 0
    if counts is not None:
        counts = _check_counts(counts, batch, index)
        c_ptr = counts.data_ptr()
    first_ptr = 0
    if isinstance(first, torch.Tensor):
        if first.shape != (batch,) or first.dtype != torch.int64 or first.get_device() != index:
            raise ValueError("first must be an int or an int64 tensor [batch] on the pages' device")
        first_dev, first = first.contiguous(), 0
        first_ptr = first_dev.data_ptr()
    else:
        first = operator.index(first)
    rotated = freq_ptr = freq_float = 0
    if frequencies is not None:
        rotated, freq_float = _check_frequencies(frequencies, dk, index)
        if not frequencies.is_contiguous():
            frequencies = frequencies.contiguous()
        freq_ptr = frequencies.data_ptr()
    p_ptr = p_sb = p_st = p_int = 0
    if positions is not None:
        if not isinstance(positions, torch.Tensor):
            raise ValueError("positions must be int64 or int32 [T] or [B, T] on the pages' device")
        positions, p_ptr, p_sb, p_st, p_int, _ = _check_positions(positions, batch, tokens, index)
    heads, q_out, q_in, q_to = 0, q, _NO_ROWS, _NO_ROWS
    if q is not None and rotated:
        heads = q_shape[1]
        q, q_out, q_in, q_to = _in_and_out(q)
    k_sb, k_sh, k_st, k_sd = k.stride()
    v_sb, v_sh, v_st, v_sd = v.stride()
    if k_sd != 1 and dk > 1:
        k = k.contiguous()
        k_sb, k_sh, k_st, _ = k.stride()
    if v_sd != 1 and dv > 1:
        v = v.contiguous()
        v_sb, v_sh, v_st, _ = v.stride()
    # Without a rotation or a rounding the keys are the caller's own.
    k_out, k_to = k, _NO_ROWS
    if rotated or dtype != k_pages.dtype:
        k_out = k_pages.new_empty(k_shape)
        k_to = k_out.data_ptr(), groups * tokens * dk, tokens * dk, dk
    if batch < 1 or tokens < 1:
        return q_out, k_out
    args = pack_rotary(*q_in, *q_to, k.data_ptr(), k_sb, k_sh, k_st, *k_to, v.data_ptr(), v_sb, v_sh, v_st,
                       k_pages.data_ptr(), kp_sp, kp_sg, kp_st, v_pages.data_ptr(), vp_sp, vp_sg, vp_st,
                       table_ptr, table_sb, n_ptr, c_ptr, freq_ptr, p_ptr, p_sb, p_st, first_ptr, first, batch, heads,
                       groups, tokens, dk, dv, rotated, _TYPES[dtype], code, int(interleaved), freq_float, p_int,
                       len_add, page, table_len, n_pages, amplitude, 1.0)
    _launch(paged_lib().logkv_paged_append, "logkv_paged_append", index, args)
    return q_out, k_out


@lru_cache(maxsize=256)
def _workspace_bytes(batch, heads, groups, tq, dk, dv, dtype, page, table_len, prefixes, prefix_len, paged_prefix):
    """Scratch of a call of these sizes."""
    args = PagedArgs(n_batch=batch, n_heads=heads, n_groups=groups, tq=tq, dk=dk, dv=dv, dtype=dtype, page=page,
                     table_len=table_len, n_prefixes=prefixes, prefix_len=prefix_len,
                     prefix_table=1 if paged_prefix else None)
    need = paged_lib().logkv_paged_workspace_bytes(bytes(args))
    if need < 0:
        raise ValueError("paged attention: " + paged_lib().logkv_last_error().decode(errors="replace"))
    return need


def _needs_gradient(prefix):
    return any(x is not None and x.requires_grad for x in (prefix.k, prefix.v, prefix.bias))


def _check_prefix(prefix, batch, groups, dk, dv, dtype, page, index):
    """(prefixes, rows or pages each, table address and stride, K and V address and strides, bias address and strides,
    its half flag, capacity in rows)."""
    _, table, pk, pv, bias, _ = prefix
    if (table is None) == (pk is None) or (pk is None) != (pv is None) or table is not None and bias is not None:
        raise ValueError("a prefix has a table of pages, or k and v rows with an optional bias")
    if table is not None:
        if table.ndim != 2:
            raise ValueError("a prefix's table must be int32 [N, n]")
        n = table.size(0)
        ptr, sb, width = _check_table(table, n, index)
        rest = n, width, ptr, sb, _NO_ROWS, _NO_ROWS, 0, _NO_STRIDES, 0, width * page
    else:
        if pk.ndim != 4 or pv.ndim != 4 or pk.shape[:3] != pv.shape[:3] or pk.size(1) != groups or pk.size(3) != dk \
                or pv.size(3) != dv or pk.dtype != dtype or pv.dtype != dtype \
                or not pk.get_device() == pv.get_device() == index:
            raise ValueError("a prefix's rows must be [N, G, capacity, d] in the pages' dtype on their device")
        n, cap = pk.size(0), pk.size(2)
        k_st, v_st = (_unit_strides(x) if cap else _NO_STRIDES for x in (pk, pv))
        if k_st is None or v_st is None:
            raise ValueError("a prefix's rows must be 16-byte aligned with contiguous features")
        b_ptr, b_st, b_half = 0, _NO_STRIDES, 0
        if bias is not None:
            if bias.shape != (n, groups, cap) or bias.get_device() != index or bias.dtype not in (torch.float32, dtype):
                raise ValueError("a prefix's bias must be [N, G, capacity] on its device, float32 or its dtype")
            b_ptr, b_st, b_half = bias.data_ptr(), bias.stride(), int(bias.dtype == dtype)
        rest = n, cap, 0, 0, (pk.data_ptr(), *k_st), (pv.data_ptr(), *v_st), b_ptr, b_st, b_half, cap
    if n < 1 or batch % n:
        raise ValueError(f"{n} prefixes do not divide a batch of {batch}")
    return rest


def log_kv_paged_attention(q, k, v, k_pages, v_pages, table, lengths, scale, *, prefix=None, visible=None, counts=None):
    """Attention of T new tokens of each sequence over its prefix, its own rows and the call's, ``[B, n_heads, T, dv]``.

    ``q [B, n_heads, T, dk]`` and the call's rows ``k [B, G, T, dk]``, ``v [B, G, T, dv]`` (post-rotation: those of
    ``log_kv_paged_append``, before or after it); ``lengths`` (an int, or int32 ``[B]``, read on the device and held to
    the table's rows) the rows of each sequence's pages before the call's. A token sees all of its prefix
    (``SharedPrefix``), all of those rows, and the call's rows up to itself, or those that ``visible`` (bool, ``[T, T]``
    or ``[B, T, T]``) shows it, as a drafted tree's ancestors and itself. ``counts`` (int32 ``[B]``, not with
    ``visible``) gives the tokens that exist per sequence of a padded batch: the others' outputs are zeros.

    Work is dealt out for rows that fill ``table`` and the prefix's capacity (lengths are not waited for): tables cut to
    the pages in use are up to four times faster than ones with much room to grow. A token that sees nothing gets zeros, and
    what hidden rows and unused slots hold (NaN, infinities) reaches no output; a table's entry outside the pool stands for a page of zeros. Queries and rows of another activation dtype are
    rounded to the pages', and the output is returned in the queries'. The pages are only read."""
    return _paged_attention(q, k, v, k_pages, v_pages, table, lengths, float(scale), prefix, visible, counts, None)


def _paged_attention(q, k, v, k_pages, v_pages, table, lengths, scale, prefix, visible, counts, prefix_in_use):
    """``prefix_in_use`` in place of the prefix's lengths: as ``_attention``'s ``in_use``."""
    refuse_tangents(q, k, v, k_pages, v_pages, *(() if prefix is None else (prefix.k, prefix.v, prefix.bias)))
    q_shape, k_shape, v_shape = q.shape, k.shape, v.shape
    if not len(q_shape) == len(k_shape) == len(v_shape) == 4:
        raise ValueError("queries and rows must be 4-dimensional")
    batch, heads, tq, dk = q_shape
    groups, dv = k_shape[1], v_shape[3]
    code, n_pages, page, k_width, v_width = _check_pages(k_pages, v_pages, groups)
    dtype, index = k_pages.dtype, k_pages.get_device()
    if k_width != dk or v_width != dv or groups < 1 or heads % groups or heads < 1 or tq < 1 or batch < 1:
        raise ValueError("pages must be [pages, G, page_size, d] with G dividing the query heads")
    if k_shape != (batch, groups, tq, dk) or v_shape != (batch, groups, tq, dv):
        raise ValueError("the call's rows must be [B, G, T, d], one per query position")
    if not v_pages.get_device() == q.get_device() == k.get_device() == v.get_device() == index:
        raise ValueError("all tensors must be on the pages' device")
    if not (0.0 < scale < math.inf):
        raise ValueError("attention scale must be positive")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or k_pages.requires_grad
                                    or v_pages.requires_grad or prefix is not None and _needs_gradient(prefix)):
        raise NotImplementedError("paged attention is for inference: it has no gradient (run it under torch.no_grad())")
    kp_st, vp_st = (_unit_strides(k_pages), _unit_strides(v_pages)) if n_pages else (_NO_STRIDES, _NO_STRIDES)
    if kp_st is None or vp_st is None:
        raise ValueError("the pages' rows must be 16-byte aligned with contiguous features")
    table_ptr, table_sb, table_len = _check_table(table, batch, index)
    vis_ptr = vis_sb = vis_st = c_ptr = 0
    if visible is not None:
        if counts is not None:
            raise ValueError("paged attention takes a mask of the call's rows or their counts")
        visible = _tree(visible, q, k_pages)
        vis_ptr, vis_sb, vis_st = visible.data_ptr(), visible.stride(0) if visible.ndim == 3 else 0, visible.stride(-2)
    elif counts is not None:
        counts = _check_counts(counts, batch, index)
        c_ptr = counts.data_ptr()
    lengths, n_ptr, n_st, len_add = _lengths(lengths, batch, table_len * page, index)
    out_dtype = q.dtype
    q_st, k_st, v_st = q.stride(), k.stride(), v.stride()
    qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (out_dtype != dtype or k.dtype != dtype or v.dtype != dtype or not q_st[3] == k_st[3] == v_st[3] == 1
            or (q_st[0] | q_st[1] | q_st[2] | k_st[0] | k_st[1] | k_st[2] | v_st[0] | v_st[1] | v_st[2]) & 7
            or (qp | kp | vp) & 15):
        q, k, v = _small_rows(q, dtype), _small_rows(k, dtype), _small_rows(v, dtype)
        q_st, k_st, v_st = q.stride(), k.stride(), v.stride()
        qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    prefixes = prefix_len = pt_ptr = pt_sb = b_ptr = b_half = pn_ptr = pn2_ptr = pn_st = pn_add = 0
    pk = pv = _NO_ROWS
    b_st, bias_scale = _NO_STRIDES, 0.0
    if prefix is not None:
        prefixes, prefix_len, pt_ptr, pt_sb, pk, pv, b_ptr, b_st, b_half, rows = _check_prefix(
            prefix, batch, groups, dk, dv, dtype, page, index)
        bias_scale = float(prefix.bias_scale)
        if not 0.0 < bias_scale < math.inf:
            raise ValueError("bias_scale must be positive")
        if prefix_in_use is not None:
            pn_ptr, pn_st, pn2_ptr, pn_add = prefix_in_use
        else:
            prefix_lengths, pn_ptr, pn_st, pn_add = _lengths(prefix.lengths, prefixes, rows, index)
    out = k_pages.new_empty((batch, heads, tq, dv))
    need = _workspace_bytes(batch, heads, groups, tq, dk, dv, code, page, table_len, prefixes, prefix_len, pt_ptr != 0)
    workspace = k_pages.new_empty(need // 2)
    o_sh = tq * dv
    args = pack_paged(
        qp, q_st[0], q_st[1], q_st[2], kp, k_st[0], k_st[1], k_st[2], vp, v_st[0], v_st[1], v_st[2],
        k_pages.data_ptr(), *kp_st, v_pages.data_ptr(), *vp_st, table_ptr, table_sb, n_ptr,
        c_ptr, vis_ptr, vis_sb, vis_st, pt_ptr, pt_sb, *pk, *pv, b_ptr, *b_st,
        pn_ptr, pn2_ptr, out.data_ptr(), heads * o_sh, o_sh, dv, batch, heads, groups, tq, dk, dv, code, page, table_len,
        n_pages, prefixes, prefix_len, n_st, len_add, pn_st, pn_add, b_half, scale, bias_scale)
    _launch(paged_lib().logkv_paged_attention, "logkv_paged_attention", index, args, workspace.data_ptr(), need)
    return out if out_dtype == dtype else out.to(out_dtype)
