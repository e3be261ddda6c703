"""One lane (batch row, KV head) of row attention in 64 bits on the device, all its queries at once, and the error that its
float32 kernels may have.

For one query, with e the error of a logit (dk products and the roundings of the scale, the bias and the exponent's
argument, each within 2^-24 of scale sum |q k| + |bias|):
 * a probability is off by a factor within 2 (2 e + 2^-20): its own logit and the sum's, exp2 within 2^-22;
 * a probability as two parts: 2^-14 (bf16: of 8 bits each), 2^-21 (fp16, and 2^-32 absolute of the largest where the
   second is subnormal);
 * a float32 sum over rows: 2^-24 per addition;
 * the output's rounding: half a step, 2^-8 (bf16) or 2^-11 (fp16, 2^-25 absolute) of the value.
All but the last scale with sum p |v|: nothing is added for values that are small beside others."""

from __future__ import annotations

import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
PARTS = {torch.bfloat16: 2.0 ** -14, torch.float16: 2.0 ** -21}


def lane(q, k, v, ck, cv, b, g, n, see, scale, bias=None, live=None):
    """(out [rep, T, dv], its bound, column sums [n + T], their relative bound) of lane (b, g) over its first n rows; ``see
    [T, T]`` (bool): the own rows that a query sees; ``live``: the tokens that exist."""
    rep, T, dk = q.size(1) // k.size(1), q.size(2), q.size(3)
    dtype, live = ck.dtype, T if live is None else live
    x = q[b, g * rep:(g + 1) * rep].double()
    keys, vals = torch.cat((ck[b, g, :n], k[b, g])).double(), torch.cat((cv[b, g, :n], v[b, g])).double()
    add = torch.zeros(n + T, dtype=torch.float64, device=q.device)
    if bias is not None:
        add[:n] = bias[b, g, :n].double()
    mask = torch.cat((torch.ones(T, n, dtype=torch.bool, device=q.device), see.to(q.device)), 1) & (add != -math.inf)
    mask[:, n + live:] = False
    mask[live:] = False
    add = torch.where(add == -math.inf, 0.0, add)
    keys, vals = (torch.where(mask.any(0)[:, None], t, 0.0) for t in (keys, vals))
    out = torch.zeros(rep, T, vals.size(1), dtype=torch.float64, device=q.device)
    bound, column = torch.zeros_like(out), torch.zeros(n + T, dtype=torch.float64, device=q.device)
    rel = 0.0
    for h in range(rep):
        s = torch.where(mask, x[h] @ keys.T * scale + add, -math.inf)
        p = torch.where(mask.any(1)[:, None], torch.softmax(s, dim=1), 0.0)
        size = torch.where(p > 0, (x[h].abs() @ keys.abs().T * scale + add.abs()), 0.0).amax(1, keepdim=True)
        logits = 2 * (2 * (dk + 8) * 2.0 ** -24 * size + 2.0 ** -20) + (n + T + 8) * 2.0 ** -24
        spread = p @ vals.abs()
        out[h] = p @ vals
        bound[h] = HALF[dtype] * out[h].abs() + (1 + HALF[dtype]) * (logits + PARTS[dtype]) * spread
        if dtype == torch.float16:
            bound[h] += 2.0 ** -24 + 2.0 ** -31 * mask.sum(1, keepdim=True) * vals.abs().amax(0)
        column += p.sum(0)
        rel = max(rel, float(logits[:live].max()) if live else 0.0)
    return out, bound, column, rel


def check_lane(got, want, bound, what=""):
    got = got.double()
    assert bool(torch.isfinite(got).all()), what
    err = (got - want).abs()
    worst = float((err / bound.clamp(min=1e-38)).max())
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"


def check_weights(w, before, column, n, cap, rel, queries, what=""):
    """A lane's weights after a call that added ``column`` [n + T] to those ``before``: sums of ``queries`` probabilities
    and the weight before in float32, the own rows' set; what lies behind them is left."""
    own = column.numel() - n
    stored = min(own, cap - n)
    want = before.double()
    want[:n] += column[:n]
    want[n:n + stored] = column[n:n + stored]
    got = w.double()
    assert bool(torch.isfinite(got).all()), what
    part = torch.zeros_like(want)
    part[:n + stored] = column[:n + stored]
    bound = (rel + (queries + 2) * 2.0 ** -24) * part + 2.0 ** -23 * want.abs() + 1e-30
    worst = float(((got - want).abs() / bound)[:n + stored].max()) if n + stored else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3f} of the weights' bound"
    assert torch.equal(w[n + stored:], before[n + stored:]), what
