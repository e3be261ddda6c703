"""Plain 64-bit forms of the row attention operators and of eviction, and the error their kernels may have.

Error of an attention output against the exact value of the same (rounded) inputs, for one query:
 * a logit: dk products summed in float32, at most (dk + 8) 2^-24 scale sum |q k| with the roundings of the scale,
   the bias and the exponent's argument, so a probability is off by a factor within 2 E + 2^-20 (the numerator's and
   the sum's logits; exp2 is within 2^-22);
 * a probability as two parts: 2^-14 relative (bf16, cut) or 2^-22 (fp16, rounded; 2^-44 absolute where the second
   part is subnormal);
 * the float32 sums over rows: each partial sum within 2^-24 per addition, at most `rows` of them;
 * bf16 values as fp16 (more than 32 queries): 2^-25 absolute below 2^-17, where a tile's largest is 2^-8 or more, and
   exact otherwise;
 * the output's rounding: half a step, 2^-8 (bf16) or 2^-11 (fp16, 2^-25 absolute) of the value.
All but the last scale with sum p |v|."""

from __future__ import annotations

import math

import torch


def reference(q, k, v, cache_k, cache_v, lengths, visible, scale, bias=None, counts=None):
    """(out, weights [B, G, capacity + T], bound of out's error, bound of the weights' relative error), float64 on the
    CPU. ``visible [B, T, T]``; hidden rows are left out before anything is computed with them."""
    q, k, v, cache_k, cache_v = (x.detach().cpu() for x in (q, k, v, cache_k, cache_v))
    B, H, T, dk = q.shape
    G, cap, dv = cache_k.size(1), cache_k.size(2), cache_v.size(3)
    rep = H // G
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[cache_k.dtype]
    parts = {torch.bfloat16: 2.0 ** -14, torch.float16: 2.0 ** -21}[cache_k.dtype]
    out = torch.zeros(B, H, T, dv, dtype=torch.float64)
    bound = torch.zeros_like(out)
    weights = torch.zeros(B, G, cap + T, dtype=torch.float64)
    rel = 0.0
    for b in range(B):
        n = min(max(int(lengths[b]), 0), cap)
        live = T if counts is None else min(max(int(counts[b]), 0), T)
        for g in range(G):
            keys = torch.cat((cache_k[b, g, :n], k[b, g, :live])).double()
            vals = torch.cat((cache_v[b, g, :n], v[b, g, :live])).double()
            add = torch.zeros(n + live, dtype=torch.float64)
            if bias is not None:
                add[:n] = bias[b, g, :n].detach().cpu().double()
            for h in range(g * rep, (g + 1) * rep):
                for t in range(live):
                    see = torch.cat((add[:n] != -math.inf, visible[b, t, :live].cpu().bool()))
                    if not see.any():
                        continue
                    kk, vv = keys[see], vals[see]
                    x = q[b, h, t].double()
                    s = kk @ x * scale + add[see]
                    p = torch.softmax(s, dim=0)
                    # Products under IEEE rules: an infinite or NaN value reaches every query that sees it.
                    out[b, h, t] = (p[:, None] * vv).sum(dim=0)
                    # Rows whose probability is zero in 64 bits take no part in the logits' size.
                    part = (p > 0) | torch.isnan(p)
                    size = float((scale * (kk[part].abs() @ x.abs()) + add[see][part].abs()).nan_to_num(0.0, 0.0, 0.0).max())
                    e = (dk + 8) * 2.0 ** -24 * size
                    factor = 2 * (2 * e + 2.0 ** -20) + parts + (len(s) + 8) * 2.0 ** -24
                    rel = max(rel, 2 * (2 * e + 2.0 ** -20) + (len(s) + 8) * 2.0 ** -24)
                    spread = p @ vv.abs()
                    bound[b, h, t] = half * out[b, h, t].abs() + (1 + half) * factor * spread
                    bound[b, h, t] += 2.0 ** -24 if cache_k.dtype == torch.float16 else (
                        2.0 ** -25 if float(vv.abs().nan_to_num(0.0, 0.0, 0.0).max()) >= 2.0 ** -8 else 0.0)
                    column = torch.zeros(n + live, dtype=torch.float64)
                    column[see] = p
                    weights[b, g, :n] += column[:n]
                    weights[b, g, cap:cap + live] += column[n:]
    return out, weights, bound, rel


def tree_mask(tokens, seed, empty=()):
    """A random tree's mask: every token sees its ancestors and itself; tokens in ``empty`` see no drafted row."""
    g = torch.Generator().manual_seed(seed)
    see = torch.zeros(tokens, tokens, dtype=torch.bool)
    for t in range(tokens):
        parent = int(torch.randint(-1, t, (1,), generator=g)) if t else -1
        if parent >= 0:
            see[t] = see[parent]
        see[t, t] = True
    for t in empty:
        see[t] = False
    return see


def check_close(got, want, bound, what=""):
    got = got.detach().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    odd = ~torch.isfinite(want)
    assert torch.equal(got[odd].nan_to_num(7.0), want[odd].nan_to_num(7.0)), what
    err = (got - want).abs()[~odd]
    worst = (err / bound[~odd].clamp(min=1e-30)).max() if err.numel() else torch.tensor(0.0)
    assert worst <= 1.0, f"{what}: {float(worst):.3f} of the bound"


def evict_reference(weights, n, keep, recent):
    """Indices that stay of one lane's first n rows."""
    if n <= keep:
        return list(range(n))
    old = n - recent
    w = weights[:old].tolist()
    rank = sorted(range(old), key=lambda i: (-math.inf if w[i] != w[i] else 0.0, 0.0 if w[i] != w[i] else -w[i], i))
    return sorted(rank[:keep - recent]) + list(range(old, n))
