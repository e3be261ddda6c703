"""Three operators over a KV cache's rows, as cases that can be timed and compared with their plain forms.

* ``tree``: attention of a tree of drafted tokens over a cache's rows and the drafted rows, each
  token seeing every cache row in use and the drafted rows that its line of the mask names;
* ``weight``: causal attention of T new tokens over a cache and themselves that adds each row's
  attention weight to the row's running sum and stores the new rows behind the cache's;
* ``evict``: the rows of a cache cut to a budget, the last ones and the heaviest others kept in order.

``run`` makes the library's calls where ``own`` is true, and computes the same in plain 32-bit torch
operations where it is false. Cache rows are ``[batch, groups, capacity, features]``; ``mass`` cases
read packed rows of the compressed cache, whose key rows carry log(mass) in the column behind the
features. Ragged batches hold sequences of different lengths.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
MOST_ROWS = 64 * 32768          # cache rows (all lanes) of the largest case
MOST_SCORES = 16 * 2048 * 32768   # (query, row) pairs of the largest case


def listed():
    return [
        # A short draft over one short conversation's compressed cache: the smallest call, latency and launches.
        dict(name="tree_1x2k_t8", kind="tree", batch=1, groups=8, heads=16, dim=128, dim_v=128, rows=2100, new=8,
             mass=True, ragged=False, dtype="bfloat16"),
        # Verification of drafted trees in eight 32K conversations over the compressed cache's packed rows.
        dict(name="tree_8x8k_t26", kind="tree", batch=8, groups=8, heads=16, dim=128, dim_v=128, rows=8782, new=26,
             mass=True, ragged=False, dtype="bfloat16"),
        # A wide tree over one long exact cache, eight query heads to a KV head.
        dict(name="tree_1x32k_t64", kind="tree", batch=1, groups=8, heads=64, dim=128, dim_v=128, rows=32768, new=64,
             mass=False, ragged=False, dtype="bfloat16"),
        # Sixteen conversations of different lengths, 64-wide heads, three to a KV head, an odd tree each.
        dict(name="tree_16x16k_t61_d64", kind="tree", batch=16, groups=4, heads=12, dim=64, dim_v=64, rows=16001,
             new=61, mass=False, ragged=True, dtype="float16"),
        # One token of one short conversation over a small budget: latency and launches.
        dict(name="weight_1x1k_t1", kind="weight", batch=1, groups=8, heads=16, dim=128, dim_v=128, rows=1024, new=1,
             ragged=False, dtype="bfloat16"),
        # One token of each of eight long conversations, nothing evicted yet.
        dict(name="weight_8x32k_t1", kind="weight", batch=8, groups=8, heads=16, dim=128, dim_v=128, rows=32768, new=1,
             ragged=False, dtype="bfloat16"),
        # Two tokens each of sixteen budgeted conversations, eight query heads to a KV head.
        dict(name="weight_16x4k_t2", kind="weight", batch=16, groups=4, heads=32, dim=96, dim_v=96, rows=4161, new=2,
             ragged=True, dtype="float16"),
        # A follow-up question over a short history: an odd chunk, 64-wide heads.
        dict(name="weight_2x4k_t333_d64", kind="weight", batch=2, groups=4, heads=8, dim=64, dim_v=64, rows=4096,
             new=333, ragged=False, dtype="bfloat16"),
        # One block of a long prompt's prefill, late in the prompt.
        dict(name="weight_1x30k_t2048", kind="weight", batch=1, groups=8, heads=16, dim=128, dim_v=128, rows=30720,
             new=2048, ragged=False, dtype="bfloat16"),
        # A decode's eviction: the rows that came since the last one.
        dict(name="evict_1x1088", kind="evict", batch=1, groups=8, dim=128, dim_v=128, rows=1088, keep=1024,
             recent=256, ragged=False, dtype="bfloat16"),
        # A model's layers as batch rows, sequences of different lengths, some below the budget.
        dict(name="evict_28x4352", kind="evict", batch=28, groups=8, dim=128, dim_v=128, rows=4352, keep=4096,
             recent=1024, ragged=True, dtype="bfloat16"),
        # Eight long prompts cut to the budget after their prefill.
        dict(name="evict_8x32k", kind="evict", batch=8, groups=8, dim=128, dim_v=128, rows=32768, keep=4096,
             recent=512, ragged=False, dtype="bfloat16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "weight", "weight", "evict"))
    groups = rng.choice((1, 2, 4, 8))
    dim, dim_v = rng.choice(((64, 64), (80, 80), (96, 96), (128, 128), (128, 128), (128, 64), (192, 128), (256, 256)))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
    ragged = rng.random() < 0.4
    batch = _log_uniform(rng, 1, 28 if kind == "evict" else 16)
    most = MOST_ROWS * 128 // (batch * groups * max(dim, dim_v))
    if kind == "evict":
        rows = _log_uniform(rng, 65, min(32768, most))
        keep = max(1, int(rows * rng.choice((0.1, 0.25, 0.5, 0.9, 0.98))))
        return dict(kind=kind, batch=batch, groups=groups, dim=dim, dim_v=dim_v, rows=rows, keep=keep,
                    recent=int(keep * rng.random() * 0.6), ragged=ragged, dtype=dtype)
    heads = groups * rng.choice((1, 2, 2, 3, 4, 5, 8))
    rows = _log_uniform(rng, 64, min(32768, most))
    new = _log_uniform(rng, 1, 128) if kind == "tree" else rng.choice((1, 1, 2, _log_uniform(rng, 3, 2048)))
    new = max(1, min(new, MOST_SCORES * 128 // (batch * heads * rows * max(dim, dim_v))))
    case = dict(kind=kind, batch=batch, groups=groups, heads=heads, dim=dim, dim_v=dim_v, rows=rows, new=new,
                ragged=ragged, dtype=dtype)
    if kind == "tree":
        case["mass"] = rng.random() < 0.5
    return case


# ----------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------

def _lengths(case):
    """Rows in use per batch row: all of ``rows``, or from ``rows`` down to about half of it."""
    batch, rows = case["batch"], case["rows"]
    return [rows - (rows // 2) * b // batch if case["ragged"] else rows for b in range(batch)]


def _tree(tokens, rng):
    """Visibility of a drafted tree: every token sees itself and its ancestors; a few trees' roots."""
    see = np.zeros((tokens, tokens), dtype=bool)
    for t in range(tokens):
        parent = -1 if t == 0 or rng.random() < 0.05 else int(rng.integers(max(0, t - 12), t))
        if parent >= 0:
            see[t] = see[parent]
        see[t, t] = True
    return see


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    batch, groups, dim, dim_v = case["batch"], case["groups"], case["dim"], case["dim_v"]
    lens = _lengths(case)

    def rows(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    state = dict(case=case, lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if case["kind"] == "evict":
        n = case["rows"]
        # Sums of attention weights: a few heavy rows, a long tail, rows that no query looked at.
        w = torch.exp(2.0 * torch.randn((batch, groups, n), generator=g, device="cuda"))
        w = w * (torch.rand((batch, groups, n), generator=g, device="cuda") >= 0.05)
        pos = torch.arange(n, device="cuda", dtype=torch.int64) + int(seed) % 1000
        return dict(state, cache_k=rows(batch, groups, n, dim), cache_v=rows(batch, groups, n, dim_v), weights=w,
                    positions=pos.expand(batch, groups, n).contiguous())
    heads, new = case["heads"], case["new"]
    cap = case["rows"] + (new if case["kind"] == "weight" else 0)
    # Queries of twice the unit scale: logits of deviation two, a few rows hold most of the weight.
    q = (2.0 * torch.randn((batch, heads, new, dim), generator=g, device="cuda")).to(dtype)
    state.update(q=q, k=rows(batch, groups, new, dim), v=rows(batch, groups, new, dim_v), scale=dim ** -0.5)
    if case["kind"] == "tree":
        rng = np.random.default_rng(int(seed))
        trees = np.stack([_tree(new, rng) for _ in range(batch if case["ragged"] else 1)])
        state["visible"] = torch.from_numpy(trees if case["ragged"] else trees[0]).cuda()
        if case["mass"]:
            width = (max(dim + 1, dim_v) + 7) // 8 * 8
            packed_k, packed_v = (torch.zeros((batch, groups, cap, width), dtype=dtype, device="cuda") for _ in range(2))
            packed_k[..., :dim] = rows(batch, groups, cap, dim)
            packed_v[..., :dim_v] = rows(batch, groups, cap, dim_v)
            mass = torch.floor(torch.rand((batch, groups, cap), generator=g, device="cuda") * 63 + 1)
            packed_k[..., dim] = torch.log(mass).to(dtype)
            state.update(cache_k=packed_k[..., :dim], cache_v=packed_v[..., :dim_v], bias=packed_k[..., dim])
            return state
        return dict(state, cache_k=rows(batch, groups, cap, dim), cache_v=rows(batch, groups, cap, dim_v), bias=None)
    # Sums over as many queries before as the call has, so that neither part hides the other.
    w = torch.exp(torch.randn((batch, groups, cap), generator=g, device="cuda")) * (heads // groups * new / case["rows"])
    return dict(state, cache_k=rows(batch, groups, cap, dim), cache_v=rows(batch, groups, cap, dim_v), weights=w)


# ----------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------

def _plain_attention(q, k, v, cache_k, cache_v, lengths, visible, scale, bias):
    """(output, weights [batch, groups, queries, capacity + new]) in 32 bits."""
    batch, heads, new, dim = q.shape
    groups, cap = cache_k.shape[1:3]
    qf = q.float().reshape(batch, groups, heads // groups * new, dim)
    s_old = torch.matmul(qf, cache_k.float().transpose(-1, -2)) * scale
    if bias is not None:
        s_old = s_old + bias.float()[:, :, None, :]
    used = torch.arange(cap, device=q.device)[None, :] < lengths[:, None]
    s_old = s_old.masked_fill(~used[:, None, None, :], -math.inf)
    s_new = torch.matmul(qf, k.float().transpose(-1, -2)) * scale
    see = visible.expand(batch, new, new)[:, None, None].expand(batch, groups, heads // groups, new, new)
    s_new = s_new.masked_fill(~see.reshape(batch, groups, -1, new), -math.inf)
    s = torch.cat((s_old, s_new), dim=-1)
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p[..., :cap], cache_v.float()) + torch.matmul(p[..., cap:], v.float())
    return out.reshape(batch, heads, new, -1).to(q.dtype), p


def _plain_tree(s):
    return _plain_attention(s["q"], s["k"], s["v"], s["cache_k"], s["cache_v"], s["lengths"], s["visible"], s["scale"],
                            s["bias"])[0]


def _plain_weight(s):
    q, cap, new = s["q"], s["cache_k"].size(2), s["q"].size(2)
    causal = torch.ones(new, new, dtype=torch.bool, device=q.device).tril()
    out, p = _plain_attention(q, s["k"], s["v"], s["cache_k"], s["cache_v"], s["lengths"], causal, s["scale"], None)
    total = p.sum(dim=2)
    s["weights"] += total[..., :cap]
    at = (s["lengths"].long()[:, None] + torch.arange(new, device=q.device)[None, :])[:, None, :].expand(-1, total.size(1), -1)
    s["weights"].scatter_(2, at, total[..., cap:])
    for cache, x in ((s["cache_k"], s["k"]), (s["cache_v"], s["v"])):
        cache.scatter_(2, at[..., None].expand(-1, -1, -1, x.size(-1)), x)
    return out, s["weights"], s["cache_k"], s["cache_v"]


def _plain_evict(s):
    case, w, lengths = s["case"], s["weights"], s["lengths"].long()
    keep, at = case["keep"], torch.arange(case["rows"], device=w.device)
    last = (at[None, :] >= (lengths - case["recent"])[:, None])[:, None, :]
    used = (at[None, :] < lengths[:, None])[:, None, :]
    key = torch.where(used, torch.where(last, torch.inf, w), -torch.inf)
    kept = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep].sort(dim=-1).values
    there = kept < lengths[:, None, None]

    def gather(x, fill):
        rest = x.shape[3:]
        got = torch.gather(x, 2, kept.reshape(*kept.shape, *(1 for _ in rest)).expand(*kept.shape, *rest))
        return torch.where(there.reshape(*kept.shape, *(1 for _ in rest)), got, fill)

    return (gather(s["cache_k"], 0.0), gather(s["cache_v"], 0.0), gather(w, 0.0), gather(s["positions"], -1),
            torch.where(there, kept, -1).int(), torch.clamp(s["lengths"], max=keep))


def run(state):
    kind = state["case"]["kind"]
    s = state
    if own:
        from logkv_amd import log_kv_evict, log_kv_tree_attention, log_kv_weight_attention

        if kind == "tree":
            return log_kv_tree_attention(s["q"], s["k"], s["v"], s["cache_k"], s["cache_v"], s["lengths"],
                                         s["visible"], s["scale"], bias=s["bias"])
        if kind == "weight":
            out = log_kv_weight_attention(s["q"], s["k"], s["v"], s["cache_k"], s["cache_v"], s["weights"],
                                          s["lengths"], s["scale"])
            return out, s["weights"], s["cache_k"], s["cache_v"]
        got = log_kv_evict(s["cache_k"], s["cache_v"], s["weights"], s["lengths"], s["case"]["keep"],
                           recent=s["case"]["recent"], positions=s["positions"])
        return got.k, got.v, got.weights, got.positions, got.kept, got.lengths
    return {"tree": _plain_tree, "weight": _plain_weight, "evict": _plain_evict}[kind](state)


# ----------------------------------------------------------------------
# What a pass cannot do without, and its result in 64 bits
# ----------------------------------------------------------------------

def work(case):
    lens, groups, dim, dim_v = _lengths(case), case["groups"], case["dim"], case["dim_v"]
    row = 2 * (dim + dim_v)
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens) * groups
        # Weights in; kept rows, their weights and positions in and out; the kept indices out.
        return {"bytes": 4 * sum(lens) * groups + kept * (2 * row + 4 + 8 + 8 + 4), "flops": 0}
    batch, heads, new = case["batch"], case["heads"], case["new"]
    bytes_ = sum(lens) * groups * row + batch * groups * new * row + batch * heads * new * 2 * (dim + dim_v)
    if case["kind"] == "tree":
        pairs = sum(n + (new + 1) / 2 for n in lens) * heads * new
        return {"bytes": bytes_ + (2 * sum(lens) * groups if case["mass"] else 0), "flops": 2 * pairs * (dim + dim_v)}
    pairs = sum(n + (new + 1) / 2 for n in lens) * heads * new
    # Weights in and out, the new rows stored.
    return {"bytes": bytes_ + 8 * sum(lens) * groups + batch * groups * new * (row + 4),
            "flops": 2 * pairs * (dim + dim_v)}


def exact(case, seed):
    s = prepare(case, seed)
    lens = _lengths(case)
    if case["kind"] == "evict":
        return _exact_evict(case, s, lens)
    batch, heads, new, groups = case["batch"], case["heads"], case["new"], case["groups"]
    per = heads // groups
    out = torch.zeros(batch, heads, new, case["dim_v"], dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["kind"] == "weight" else None
    for b in range(batch):
        n = lens[b]
        if case["kind"] == "weight":
            hidden = torch.ones(new, new, dtype=torch.bool, device="cuda").triu(1)
        else:
            see = s["visible"]
            hidden = ~(see[b] if see.dim() == 3 else see)
        for g in range(groups):
            keys = torch.cat((s["cache_k"][b, g, :n], s["k"][b, g])).double()
            vals = torch.cat((s["cache_v"][b, g, :n], s["v"][b, g])).double()
            for h in range(g * per, (g + 1) * per):
                logit = (s["q"][b, h].double() @ keys.T) * s["scale"]
                if s.get("bias") is not None:
                    logit[:, :n] += s["bias"][b, g, :n].double()
                logit[:, n:][hidden] = -math.inf
                p = torch.softmax(logit, dim=-1)
                out[b, h] = p @ vals
                if weights is not None:
                    column = p.sum(dim=0)
                    if h == g * per:
                        weights[b, g, n:n + new] = 0.0
                    weights[b, g, :n + new] += column
    return out if weights is None else (out, weights, None, None)


def _exact_evict(case, s, lens):
    keep, recent = case["keep"], case["recent"]
    w = s["weights"].cpu().numpy()
    kept = np.full((case["batch"], case["groups"], keep), -1, dtype=np.int64)
    for b, n in enumerate(lens):
        for g in range(case["groups"]):
            if n <= keep:
                kept[b, g, :n] = np.arange(n)
                continue
            old = n - recent
            heavy = np.lexsort((np.arange(old), -w[b, g, :old].astype(np.float64)))[:keep - recent]
            kept[b, g] = np.concatenate((np.sort(heavy), np.arange(old, n)))
    idx = torch.from_numpy(kept).cuda()
    there, safe = idx >= 0, idx.clamp(min=0)

    def rows(x):
        return (torch.gather(x, 2, safe[..., None].expand(-1, -1, -1, x.size(-1))) * there[..., None]).double()

    return (rows(s["cache_k"]), rows(s["cache_v"]), (torch.gather(s["weights"], 2, safe) * there).double(), None, None,
            None)
