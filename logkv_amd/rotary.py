"""Rotary positions: queries and keys turned by their tokens' positions, for training and inference.

A model rotates before it calls this package's caches (they take post-RoPE queries and keys beside the pre-RoPE
keys that routing uses); ``log_kv_rotary`` is that step in one launch, with angles formed in 64 bits instead of read
from a table, and ``rotary_tables`` gives the tables of the same frequencies that ``LogStructuredKVCache`` takes
(``cos_cache``, ``sin_cache``; half layout). The reference rotates in torch (litgpt/model.py:918-925).
"""

from __future__ import annotations

import math
import operator

import torch

from ._lib import check_activation_dtype, refuse_tangents, require_device
from ._paged import F32, ROTARY_SIGNS, pack_rotary_rest, pack_rotary_rows, paged_lib
from ._rows import BF16, F16
from .row_attention import _launch

_TYPES = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}
_NO_ROWS = (0, 0, 0, 0)
MAX_WIDTH = 512


def rotary_frequencies(dim, base=10000.0, *, scaling=None, device="cuda"):
    """(frequencies, amplitude) of ``dim`` rotated features: radians per position, float64 ``[dim / 2]`` on ``device``,
    and the factor of the rotated values.

    ``scaling`` fits them to contexts longer than a model was trained on: a dict with ``kind`` and ``factor``;

    * ``"linear"``: every frequency divided by the factor;
    * ``"wavelength"``: with ``original_max_seq_len`` n, ``low_freq_factor`` l and ``high_freq_factor`` h: wavelengths
      above n / l divided by the factor, below n / h kept, interpolated between;
    * ``"yarn"``: with ``original_max_seq_len`` and optionally ``beta_fast`` (32), ``beta_slow`` (1): pairs that turn
      more than beta_fast times over that length kept, fewer than beta_slow times divided, a ramp over the pairs
      between; amplitude ``0.1 ln(factor) + 1`` or ``attention_factor``."""
    if dim < 2 or dim % 2 or dim > MAX_WIDTH:
        raise ValueError(f"rotated features must be an even number up to {MAX_WIDTH}")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError("the rotary base must be finite and above 1")
    freq = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    amplitude = 1.0
    if scaling is not None:
        given = dict(scaling)
        kind, factor = given.pop("kind", None), float(given.pop("factor", 0.0))
        if not (math.isfinite(factor) and factor > 0.0):
            raise ValueError("scaling needs a positive factor")
        try:
            if kind == "linear":
                freq = freq / factor
            elif kind == "wavelength":
                low, high = float(given.pop("low_freq_factor")), float(given.pop("high_freq_factor"))
                turns = _length(given) * freq / (2 * math.pi)
                if not 0.0 < low < high < math.inf:
                    raise ValueError("low_freq_factor must be positive and below high_freq_factor")
                keep = ((turns - low) / (high - low)).clamp(0, 1)
                freq = freq * (keep + (1 - keep) / factor)
            elif kind == "yarn":
                n, fast, slow = _length(given), float(given.pop("beta_fast", 32.0)), float(given.pop("beta_slow", 1.0))
                if not 0.0 < slow < fast < math.inf:
                    raise ValueError("beta_slow must be positive and below beta_fast")

                def pair(turns):   # the pair that turns so often over the original length
                    return dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

                lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
                ramp = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
                freq = freq * (1 - ramp + ramp / factor)
                amplitude = float(given.pop("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0))
                if not math.isfinite(amplitude):
                    raise ValueError("attention_factor must be finite")
            else:
                raise ValueError(f"unknown scaling {kind!r}: 'linear', 'wavelength' or 'yarn'")
        except KeyError as e:
            raise ValueError(f"scaling {kind!r} needs {e.args[0]}") from None
        if given:
            raise ValueError(f"scaling {kind!r} takes no {', '.join(sorted(given))}")
    return freq.to(device), amplitude


def _length(given):
    n = float(given.pop("original_max_seq_len"))
    if not (math.isfinite(n) and n >= 1.0):
        raise ValueError("original_max_seq_len must be at least 1")
    return n


def rotary_tables(frequencies, n, *, amplitude=1.0, dtype=torch.float32):
    """(cos, sin) ``[n, dim]`` of positions 0 .. n - 1 in the half layout, as ``LogStructuredKVCache`` takes them: each
    the 64-bit value rounded once."""
    angles = torch.outer(torch.arange(n, dtype=torch.float64, device=frequencies.device), frequencies.double())
    angles = torch.cat((angles, angles), dim=-1)
    return (amplitude * torch.cos(angles)).to(dtype), (amplitude * torch.sin(angles)).to(dtype)


def _in_and_out(x):
    """(rows with contiguous features, new ones in their dimension order, addresses and strides of both: 0 of none)."""
    y = torch.empty_like(x)
    sb, sh, st, sd = tb, th, tt, td = x.stride()
    if not x.is_contiguous():
        tb, th, tt, td = y.stride()
    if (sd != 1 or td != 1) and x.size(3) != 1:
        x = x.contiguous()
        y = torch.empty_like(x)
        (sb, sh, st, _), (tb, th, tt, _) = x.stride(), y.stride()
    if not x.numel():
        return x, y, _NO_ROWS, _NO_ROWS
    return x, y, (x.data_ptr(), sb, sh, st), (y.data_ptr(), tb, th, tt)


def _check_frequencies(frequencies, dim, index):
    """(address, rotated features, whether float32)."""
    shape, dtype = frequencies.shape, frequencies.dtype
    if (len(shape) != 1 or dtype is not torch.float64 and dtype is not torch.float32
            or frequencies.get_device() != index or 2 * shape[0] > dim):
        raise ValueError("frequencies must be float64 or float32 [rotated features / 2] on the rows' device, "
                         f"for up to {dim} features")
    if frequencies.requires_grad:
        raise NotImplementedError("frequencies have no gradient")
    return 2 * shape[0], int(dtype is torch.float32)


def _check_positions(positions, batch, tokens, index):
    """(tensor or None, address, strides, whether int32, first position)."""
    if not isinstance(positions, torch.Tensor):
        return None, 0, 0, 0, 0, operator.index(positions)
    shape = positions.shape
    if (not (shape == (tokens,) or shape == (batch, tokens)) or positions.get_device() != index
            or positions.dtype not in (torch.int64, torch.int32)):
        raise ValueError("positions must be an int, or int64 or int32 [T] or [B, T] on the rows' device")
    sb, st = (0, positions.stride(0)) if len(shape) == 1 else positions.stride()
    return positions, positions.data_ptr(), sb, st, int(positions.dtype == torch.int32), 0


def _plan(shape, groups, dtype, index, frequencies, positions, interleaved, amplitude):
    """What a launch needs beside its rows and its sign, with the tensors that it points into."""
    batch, heads, tokens, dim = shape
    rotated, freq_float = _check_frequencies(frequencies, dim, index)
    if not frequencies.is_contiguous():
        frequencies = frequencies.contiguous()
    positions, p_ptr, p_sb, p_st, p_int, first = _check_positions(positions, batch, tokens, index)
    rest = pack_rotary_rest(*_NO_ROWS, *_NO_ROWS, *_NO_ROWS, 0, 0, 0, 0, frequencies.data_ptr(), p_ptr, p_sb, p_st, 0, first,
                            batch, heads, groups, tokens, dim, 0, rotated, _TYPES[dtype], 0, int(interleaved), freq_float,
                            p_int, 0, 0, 0, 0, amplitude)
    return rest, frequencies, positions


def _rotate(q, k, rest, sign, index):
    """The launch; q or k may be None."""
    q_in = q_to = k_in = k_to = _NO_ROWS
    q_out = k_out = None
    if q is not None:
        q, q_out, q_in, q_to = _in_and_out(q)
    if k is not None:
        k, k_out, k_in, k_to = _in_and_out(k)
    if q_in[0] or k_in[0]:
        args = pack_rotary_rows(*q_in, *q_to, *k_in, *k_to) + rest + ROTARY_SIGNS[sign]
        _launch(paged_lib().logkv_rotary, "logkv_rotary", index, args)
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """The rotation as a function of the rows; its gradient is the rotation back. ``state`` is what a launch needs beside
    them: (arguments, device, frequencies, positions, their versions). The tensors are held here, not saved through
    autograd, whose way there and back takes as long as a launch."""

    @staticmethod
    def forward(ctx, q, k, state, sign):
        ctx.set_materialize_grads(False)
        ctx.state, ctx.sign = state, sign
        out = _rotate(q, k, state[0], sign, state[1])
        need_q, need_k, _, _ = ctx.needs_input_grad
        if not (need_q and need_k):
            ctx.mark_non_differentiable(*(y for y, need in zip(out, (need_q, need_k)) if y is not None and not need))
        return out

    @staticmethod
    def backward(ctx, dq, dk):
        state, sign = ctx.state, -ctx.sign
        rest, index, frequencies, positions, versions = state
        if versions != _versions(frequencies, positions):
            raise RuntimeError("the frequencies or positions of a rotation have been modified in place before its gradient")
        if torch.is_grad_enabled():      # the gradient has a graph of its own
            return *_Rotary.apply(dq, dk, state, sign), None, None
        return *_rotate(dq, dk, rest, sign, index), None, None


def _versions(frequencies, positions):
    return frequencies._version, 0 if positions is None else positions._version


def log_kv_rotary(q, k, frequencies, positions=0, *, interleaved=False, amplitude=1.0):
    """(q, k) rotated by their tokens' positions: pair i of a head's first ``2 n`` features turned by ``position *
    frequencies[i]`` and scaled by ``amplitude``, its other features as they are.

    ``q [B, n_heads, T, d]`` and ``k [B, G, T, d]`` (or None) in one of bfloat16, float16 or float32, of any strides;
    ``frequencies [n]`` in radians per position, float64 or float32 (``rotary_frequencies``); ``positions`` the first
    token's (an int), or int64 or int32 ``[T]`` or ``[B, T]``. Pairs are features ``(i, i + n)``, or ``(2 i, 2 i + 1)``
    with ``interleaved``. Angles are formed in 64 bits, products in float32, rounded once. New tensors in the inputs'
    dimension order; differentiable in q and k any number of times (captured into a HIP graph, like any backward pass, over
    leaves that no graph of an eager call still holds). Dual tensors (forward mode) are refused."""
    refuse_tangents(q, k, frequencies)
    shape, dtype, index, groups = q.shape, q.dtype, q.get_device(), 0
    if len(shape) != 4:
        raise ValueError("q and k must be [B, heads, T, d] of one batch, length and width")
    if k is not None:
        other = k.shape
        if len(other) != 4 or other[0] != shape[0] or other[2] != shape[2] or other[3] != shape[3]:
            raise ValueError("q and k must be [B, heads, T, d] of one batch, length and width")
        if k.dtype is not dtype or k.get_device() != index:
            raise ValueError("q and k must be of one dtype on one device")
        groups = other[1]
    check_activation_dtype(dtype)
    if index < 0:
        require_device(q, "q")
    if not 1 <= shape[3] <= MAX_WIDTH:
        raise ValueError(f"head widths must be in [1, {MAX_WIDTH}]")
    amplitude = float(amplitude)
    if not math.isfinite(amplitude):
        raise ValueError("amplitude must be finite")
    rest, frequencies, positions = _plan(shape, groups, dtype, index, frequencies, positions, interleaved, amplitude)
    if torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad):
        state = rest, index, frequencies, positions, _versions(frequencies, positions)
        return _Rotary.apply(q, k, state, 1.0)
    return _rotate(q, k, rest, 1.0, index)
