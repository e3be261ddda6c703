"""Plain 64-bit forms of the rotation, of appends to a paged cache and of attention over one, and their kernels' errors.

Error of a rotated feature: the angle is reduced to a turn in 64 bits and rounded to float32 (2^-26 of a turn,
2 pi 2^-26 < 2^-23 radians), its sine and cosine are within 4 ulp (2^-22), the amplitude's product and the two products
with the pair add 2^-24 each: together within 2^-21 amplitude (|a| + |b|). The output's rounding: half a step, 2^-8 (bf16),
2^-11 (fp16, 2^-25 absolute below its normals) or 2^-24 (float32) of the value."""

from __future__ import annotations

import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rotate(x, frequencies, positions, interleaved=False, amplitude=1.0, sign=1.0, to=None):
    """(y, bound) of ``x [B, H, T, d]`` at ``positions [B, T]``, float64 on the CPU; ``to``: the output's dtype."""
    half = HALF[x.dtype if to is None else to]
    x, f = x.detach().cpu().double(), frequencies.detach().cpu().double()
    n = f.numel()
    angles = sign * positions.cpu().double()[:, None, :, None] * f
    y, size = x.clone(), torch.zeros_like(x)
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        c, s = amplitude * torch.cos(angles[..., i]), amplitude * torch.sin(angles[..., i])
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = abs(amplitude) * (x[..., a].abs() + x[..., b].abs())
    return y, half * y.abs() + (1 + half) * 2.0 ** -21 * size + 2.0 ** -25 * (half == 2.0 ** -11)


def dense(pages, table, lengths, cap):
    """The rows of each sequence, ``[B, G, cap, d]``, zeros behind its last and for pages outside the pool (CPU)."""
    pages, table = pages.detach().cpu(), table.cpu()
    page = pages.size(2)
    out = torch.zeros(table.size(0), pages.size(1), cap, pages.size(3), dtype=pages.dtype)
    for b, n in enumerate(lengths):
        for i in range(min(n, cap)):
            at = int(table[b, i // page])
            if 0 <= at < pages.size(0):
                out[b, :, i] = pages[at, :, i % page]
    return out


def joined(own, prefix, batch):
    """(rows ``[B, G, cap, d]``, lengths) of each sequence's prefix followed by its own rows, from (rows, lengths) pairs."""
    rows, lengths = own
    if prefix is None:
        return rows, list(lengths)
    shared, sizes = prefix
    run = batch // shared.size(0)
    total = [sizes[b // run] + lengths[b] for b in range(batch)]
    out = torch.zeros(batch, rows.size(1), max(max(total), 1), rows.size(3), dtype=rows.dtype)
    for b in range(batch):
        p = sizes[b // run]
        out[b, :, :p] = shared[b // run, :, :p]
        out[b, :, p:total[b]] = rows[b, :, :lengths[b]]
    return out, total


def joined_bias(bias, sizes, lengths, cap, scale=1.0):
    """The bias of ``joined`` rows: the prefix's times ``scale``, zeros behind it."""
    batch, run = len(lengths), len(lengths) // bias.size(0)
    out = torch.zeros(batch, bias.size(1), cap, dtype=torch.float64)
    for b in range(batch):
        p = sizes[b // run]
        out[b, :, :p] = bias[b // run, :, :p].detach().cpu().double() * scale
    return out


def pool(batch, groups, dk, dv, page, sizes, dtype, seed, device, spare=2, fill=None):
    """(k_pages, v_pages, table) of random rows in random pages; entries behind a sequence's last page are -1."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in sizes]
    order = torch.randperm(sum(need) + spare, generator=g).int()
    table = torch.full((batch, max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pages = [torch.randn(sum(need) + spare, groups, page, d, generator=g).to(dtype) for d in (dk, dv)]
    if fill is not None:      # slots that hold no row
        for b, n in enumerate(sizes):
            if n % page:
                for x in pages:
                    x[table[b, n // page], :, n % page:] = fill
        for x in pages:
            x[order[at:].long()] = fill
    return (*(x.to(device) for x in pages), table.to(device))


def inverse(f, n):
    """Frequencies of ``n`` pairs for the tests."""
    return f ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) if n else torch.zeros(0, dtype=torch.float64)


def within(got, want, bound, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    odd = ~torch.isfinite(want)
    assert torch.equal(got[odd].nan_to_num(7.0), want[odd].nan_to_num(7.0)), what
    err = ((got - want).abs() / bound.clamp(min=1e-30))[~odd]
    worst = float(err.max()) if err.numel() else 0.0
    assert worst <= 1.0 and not math.isnan(worst), f"{what}: {worst:.3f} of the bound"
