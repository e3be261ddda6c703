"""Three operators around an exact cache in pages, as cases that can be timed and compared with their plain forms.

* ``rotary``: queries and keys rotated by their positions, both layouts, whole heads or a part, and the gradients;
* ``append``: new keys and values stored in a paged cache, keys (and the queries beside them) rotated on the way;
* ``prefix``: attention of a batch whose sequences share long prefixes: every prefix's rows are read once for all
  of its sequences, then each sequence's own rows in their pages, and the call's rows causally.

``run`` makes the library's calls where ``own`` is true, and computes the same in plain 32-bit torch operations
(angles in 64 bits) where it is false. Pages are ``[pages, groups, page_size, features]``; a table holds each
sequence's page numbers, -1 where it has no page. ``mass`` cases share a prefix of packed rows of the compressed
cache, whose key rows carry log(mass) in the column behind the features.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
MOST_VALUES = 16384 * 48 * 128        # rotated values of the largest case
MOST_ROWS = 8 * 4096 * 8              # appended rows (all groups) of the largest case
MOST_PAIRS = 8 * 16 * 256 * 33000     # (query, row) pairs of the largest case
MOST_OWN = 64 * 8 * 2200              # rows in pages (all groups) of the largest case


def listed():
    return [
        # The next token of one conversation: the smallest call, latency and launches.
        dict(name="rotary_1x1", kind="rotary", batch=1, heads=16, groups=8, dim=128, rotated=128, new=1, first=32000,
             stretch=1.0, interleaved=False, train=False, dtype="bfloat16"),
        # A training step's chunk: the rotation and its gradients.
        dict(name="rotary_2x1024_train", kind="rotary", batch=2, heads=16, groups=8, dim=128, rotated=128, new=1024,
             first=0, stretch=1.0, interleaved=False, train=True, dtype="bfloat16"),
        # A long prompt of odd length, far positions, neighbouring pairs in a part of the head, positions stretched.
        dict(name="rotary_1x16001_part", kind="rotary", batch=1, heads=32, groups=8, dim=128, rotated=64, new=16001,
             first=100000, stretch=4.0, interleaved=True, train=False, dtype="float16"),
        # The next token of one conversation: latency and launches.
        dict(name="append_1x1", kind="append", batch=1, heads=16, groups=8, dim=128, dim_v=128, rotated=128, new=1,
             rows=2100, page=64, first=0, stretch=1.0, interleaved=False, ragged=False, dtype="bfloat16"),
        # A decode step of many conversations of different lengths.
        dict(name="append_64x1", kind="append", batch=64, heads=32, groups=8, dim=128, dim_v=128, rotated=128, new=1,
             rows=2000, page=16, first=16384, stretch=1.0, interleaved=False, ragged=True, dtype="bfloat16"),
        # Follow-up questions of odd, different lengths; wide keys of which a part is rotated.
        dict(name="append_12x333_part", kind="append", batch=12, heads=16, groups=4, dim=192, dim_v=128, rotated=64,
             new=333, rows=1601, page=32, first=0, stretch=8.0, interleaved=True, ragged=True, dtype="float16"),
        # Prompts of a batch written as a whole.
        dict(name="append_8x4096", kind="append", batch=8, heads=16, groups=8, dim=128, dim_v=128, rotated=128,
             new=4096, rows=0, page=64, first=0, stretch=1.0, interleaved=False, ragged=False, dtype="bfloat16"),
        # A few short answers behind one instruction: latency and launches.
        dict(name="prefix_4x2k_t1", kind="prefix", batch=4, prefixes=1, heads=16, groups=8, dim=128, dim_v=128,
             shared=2048, rows=200, new=1, page=64, mass=False, ragged=True, dtype="bfloat16"),
        # Many answers to one long prompt, four query heads to a KV head.
        dict(name="prefix_64x16k_t1", kind="prefix", batch=64, prefixes=1, heads=32, groups=8, dim=128, dim_v=128,
             shared=16384, rows=2000, new=1, page=16, mass=False, ragged=True, dtype="bfloat16"),
        # Two prompts with twelve answers each, seven tokens a step, 64-wide heads, three to a KV head.
        dict(name="prefix_24x8k_t7_d64", kind="prefix", batch=24, prefixes=2, heads=12, groups=4, dim=64, dim_v=64,
             shared=8001, rows=901, new=7, page=32, mass=False, ragged=True, dtype="float16"),
        # Answers over one compressed 32K document.
        dict(name="prefix_32x8782_mass", kind="prefix", batch=32, prefixes=1, heads=16, groups=8, dim=128, dim_v=128,
             shared=8782, rows=512, new=1, page=64, mass=True, ragged=True, dtype="bfloat16"),
        # Questions about one long document, each read as a whole.
        dict(name="prefix_8x32k_t256", kind="prefix", batch=8, prefixes=1, heads=16, groups=8, dim=128, dim_v=128,
             shared=32768, rows=0, new=256, page=64, mass=False, ragged=False, dtype="bfloat16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rotary", "append", "prefix", "prefix"))
    groups = rng.choice((1, 2, 4, 8))
    heads = groups * rng.choice((1, 2, 2, 3, 4, 5, 8))
    dim, dim_v = rng.choice(((64, 64), (80, 80), (96, 96), (128, 128), (128, 128), (128, 64), (192, 128), (256, 256)))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
    batch = _log_uniform(rng, 1, 64)
    turn = dict(rotated=2 * rng.choice((dim // 2, dim // 2, dim // 4, dim // 8 + 1)), interleaved=rng.random() < 0.4,
                first=rng.choice((0, 0, _log_uniform(rng, 1, 1000000))), stretch=rng.choice((1.0, 1.0, 4.0, 32.0)))
    if kind == "rotary":
        new = _log_uniform(rng, 1, max(1, min(32768, MOST_VALUES // (2 * batch * (heads + groups) * dim))))
        return dict(kind=kind, batch=batch, heads=heads, groups=groups, dim=dim, new=new, train=rng.random() < 0.4,
                    dtype=rng.choice((dtype, dtype, "float32")), **turn)
    ragged, page = rng.random() < 0.5, rng.choice((16, 32, 64, 128, 256))
    if kind == "append":
        new = _log_uniform(rng, 1, max(1, min(4096, MOST_ROWS // (batch * groups) * 128 // dim)))
        return dict(kind=kind, batch=batch, heads=heads, groups=groups, dim=dim, dim_v=dim_v, new=new,
                    rows=rng.choice((0, _log_uniform(rng, 1, 2048))), page=page, ragged=ragged, dtype=dtype, **turn)
    prefixes = rng.choice((1, 1, 2, 3))
    batch = prefixes * _log_uniform(rng, 1, 64 // prefixes)
    rows = min(rng.choice((0, _log_uniform(rng, 1, 2048), _log_uniform(rng, 1, 2048))), MOST_OWN // (batch * groups))
    shared = _log_uniform(rng, 16, 32768)
    new = rng.choice((1, 1, _log_uniform(rng, 2, 16), _log_uniform(rng, 2, 256)))
    new = max(1, min(new, MOST_PAIRS * 128 // (batch * heads * (shared + rows + 256) * max(dim, dim_v))))
    return dict(kind=kind, batch=batch, prefixes=prefixes, heads=heads, groups=groups, dim=dim, dim_v=dim_v,
                shared=shared, rows=rows, new=new, page=page, mass=rng.random() < 0.3, ragged=ragged, dtype=dtype)


# ----------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------

def _lengths(case):
    """Rows in use per sequence: all of ``rows``, or from ``rows`` down to about half of it."""
    batch, rows = case["batch"], case["rows"]
    return [rows - (rows // 2) * b // batch if case["ragged"] else rows for b in range(batch)]


def _counts(case):
    """New tokens per sequence of a padded batch."""
    batch, new = case["batch"], case["new"]
    return [new - (new // 2) * b // batch if case["ragged"] else new for b in range(batch)]


def _tables(sizes, page, rng):
    """(tables of page numbers, -1 where a sequence has no page; pages in all), pages in random order."""
    need = [-(-n // page) for n in sizes]
    order = torch.randperm(sum(need) + 3, generator=rng, device="cuda").int()
    table = torch.full((len(sizes), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    batch, heads, groups, dim, new = (case[n] for n in ("batch", "heads", "groups", "dim", "new"))

    def rows(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    state = dict(case=case, q=rows(batch, heads, new, dim), k=rows(batch, groups, new, dim))
    if case["kind"] != "prefix":
        half = case["rotated"] // 2
        state["frequencies"] = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half) / case["stretch"]
    if case["kind"] == "rotary":
        state["positions"] = torch.arange(new, device="cuda") + (case["first"] + int(seed) % 97)
        if case["train"]:
            state.update(grad_q=rows(batch, heads, new, dim), grad_k=rows(batch, groups, new, dim))
            state["q"].requires_grad_(), state["k"].requires_grad_()
        return state
    lens, page, dim_v = _lengths(case), case["page"], case["dim_v"]
    state.update(v=rows(batch, groups, new, dim_v), lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if case["kind"] == "append":
        counts = _counts(case)
        table, pages = _tables([n + c for n, c in zip(lens, counts)], page, g)
        state.update(counts=torch.tensor(counts, dtype=torch.int32, device="cuda") if case["ragged"] else None,
                     table=table)
    else:
        # Queries of twice the unit scale: logits of deviation two, a few rows hold most of the weight.
        state["q"] *= 2.0
        shared, prefixes = case["shared"], case["prefixes"]
        state["prefix_lengths"] = torch.tensor([shared - (shared // 3) * i // prefixes for i in range(prefixes)],
                                               dtype=torch.int32, device="cuda")
        sizes = [max(n, 1) for n in lens]
        table, pages = _tables(sizes if case["mass"] else sizes + [shared] * prefixes, page, g)
        state.update(table=table[:batch, :-(-max(sizes) // page)].contiguous(), scale=dim ** -0.5, prefix_table=None,
                     prefix_k=None, prefix_v=None, prefix_bias=None)
        if case["mass"]:
            width = (max(dim + 1, dim_v) + 7) // 8 * 8
            packed_k, packed_v = (torch.zeros((prefixes, groups, shared, width), dtype=dtype, device="cuda") for _ in range(2))
            packed_k[..., :dim] = rows(prefixes, groups, shared, dim)
            packed_v[..., :dim_v] = rows(prefixes, groups, shared, dim_v)
            mass = torch.floor(torch.rand((prefixes, groups, shared), generator=g, device="cuda") * 63 + 1)
            packed_k[..., dim] = torch.log(mass).to(dtype)
            state.update(prefix_k=packed_k[..., :dim], prefix_v=packed_v[..., :dim_v], prefix_bias=packed_k[..., dim])
        else:
            state["prefix_table"] = table[batch:, :-(-shared // page)].contiguous()
    return dict(state, k_pages=rows(pages, groups, page, dim), v_pages=rows(pages, groups, page, dim_v))


# ----------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------

def _plain_rotate(x, angles, interleaved, back=False):
    """x ``[B, H, T, d]`` in 32 bits, rotated by angles ``[B or 1, T, r / 2]``; ``back``: by their negatives."""
    cos, sin = torch.cos(angles).float()[:, None], torch.sin(angles).float()[:, None]
    if back:
        sin = -sin
    half, x = angles.size(-1), x.float()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _plain_rotary(s):
    case = s["case"]
    angles = (s["positions"].double()[:, None] * s["frequencies"])[None]
    with torch.no_grad():
        out = tuple(_plain_rotate(x, angles, case["interleaved"]).to(x.dtype) for x in (s["q"], s["k"]))
        if case["train"]:
            out += tuple(_plain_rotate(x, angles, case["interleaved"], back=True).to(x.dtype)
                         for x in (s["grad_q"], s["grad_k"]))
    return out


def _plain_append(s):
    case, table, page = s["case"], s["table"].long(), s["case"]["page"]
    at = s["lengths"].long()[:, None] + torch.arange(case["new"], device=table.device)
    angles = (at + case["first"]).double()[..., None] * s["frequencies"]
    q, k = (_plain_rotate(x, angles, case["interleaved"]).to(x.dtype) for x in (s["q"], s["k"]))
    there = torch.ones_like(at, dtype=torch.bool)
    if s["counts"] is not None:
        there = torch.arange(case["new"], device=table.device) < s["counts"][:, None]
    b, t = there.nonzero(as_tuple=True)
    pages, slots = table[b, at[b, t] // page], at[b, t] % page
    s["k_pages"][pages, :, slots] = k[b, :, t]
    s["v_pages"][pages, :, slots] = s["v"][b, :, t]
    return q, k, s["k_pages"], s["v_pages"]


def _plain_prefix(s):
    case, q = s["case"], s["q"]
    batch, heads, new, dim = q.shape
    groups, prefixes = case["groups"], case["prefixes"]
    per, share = heads // groups, batch // prefixes

    def paged(pages, table):
        x = pages[table.long().clamp(min=0)].float()      # [n, pages, groups, page, d]
        return x.transpose(1, 2).flatten(2, 3)

    if s["prefix_table"] is not None:
        kp, vp = paged(s["k_pages"], s["prefix_table"]), paged(s["v_pages"], s["prefix_table"])
    else:
        kp, vp = s["prefix_k"].float(), s["prefix_v"].float()
    ko, vo = (torch.cat((paged(s[n + "_pages"], s["table"]), s[n].float()), dim=2) for n in "kv")

    def by_prefix(x):      # [B, G, per * T, d] -> [N, G, share * per * T, d], the queries that share a prefix's rows
        return x.reshape(prefixes, share, groups, per * new, -1).transpose(1, 2).flatten(2, 3)

    def by_sequence(x):
        return x.reshape(prefixes, groups, share, per * new, -1).transpose(1, 2).flatten(0, 1)

    qf = q.float().reshape(batch, groups, per * new, dim)
    sp = torch.matmul(by_prefix(qf), kp.transpose(-1, -2)) * s["scale"]
    if s["prefix_bias"] is not None:
        sp = sp + s["prefix_bias"].float()[:, :, None, :]
    used = torch.arange(kp.size(2), device=q.device)[None, :] < s["prefix_lengths"][:, None]
    sp = sp.masked_fill(~used[:, None, None, :], -math.inf)
    so = torch.matmul(qf, ko.transpose(-1, -2)) * s["scale"]
    cap = ko.size(2) - new
    used = (torch.arange(cap, device=q.device)[None, :] < s["lengths"][:, None])[:, None, :].expand(batch, new, cap)
    causal = torch.ones(new, new, dtype=torch.bool, device=q.device).tril()
    see = torch.cat((used, causal.expand(batch, new, new)), dim=-1)[:, None, None]
    so = so.masked_fill(~see.expand(batch, groups, per, new, -1).reshape(batch, groups, per * new, -1), -math.inf)
    m = torch.maximum(by_sequence(sp.amax(dim=-1, keepdim=True)), so.amax(dim=-1, keepdim=True))
    sp, so = torch.exp(sp - by_prefix(m)), torch.exp(so - m)
    total = by_sequence(sp.sum(dim=-1, keepdim=True)) + so.sum(dim=-1, keepdim=True)
    out = (by_sequence(torch.matmul(sp, vp)) + torch.matmul(so, vo)) / total
    return out.reshape(batch, heads, new, -1).to(q.dtype)


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append, "prefix": _plain_prefix}[case["kind"]](s)
    import logkv_amd

    if case["kind"] == "rotary":
        q, k = logkv_amd.log_kv_rotary(s["q"], s["k"], s["frequencies"], s["positions"], interleaved=case["interleaved"])
        if not case["train"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["grad_q"], s["grad_k"]))
        return q.detach(), k.detach(), dq, dk
    if case["kind"] == "append":
        q, k = logkv_amd.log_kv_paged_append(
            s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], q=s["q"],
            frequencies=s["frequencies"], first=case["first"], interleaved=case["interleaved"], counts=s["counts"])
        return q, k, s["k_pages"], s["v_pages"]
    prefix = logkv_amd.SharedPrefix(s["prefix_lengths"], table=s["prefix_table"], k=s["prefix_k"], v=s["prefix_v"],
                                    bias=s["prefix_bias"])
    return logkv_amd.log_kv_paged_attention(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"],
                                            s["lengths"], s["scale"], prefix=prefix)


# ----------------------------------------------------------------------
# What a pass cannot do without, and its result in 64 bits
# ----------------------------------------------------------------------

def work(case):
    batch, heads, groups, dim, new = (case[n] for n in ("batch", "heads", "groups", "dim", "new"))
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "rotary":
        values = batch * new * (heads + groups)
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * size * values * dim, "flops": passes * 3 * values * case["rotated"]}
    dim_v = case["dim_v"]
    if case["kind"] == "append":
        stored = sum(_counts(case)) * groups
        # Queries in and out, keys in and out, and what is stored.
        return {"bytes": size * (2 * batch * new * (heads + groups) * dim + stored * (dim + 2 * dim_v)),
                "flops": 3 * batch * new * (heads + groups) * case["rotated"]}
    lens, shared, prefixes = _lengths(case), case["shared"], case["prefixes"]
    prefix = [shared - (shared // 3) * i // prefixes for i in range(prefixes)]
    rows = (sum(lens) + sum(prefix) + batch * new) * groups
    pairs = heads * new * (sum(lens) + batch // prefixes * sum(prefix) + batch * (new + 1) / 2)
    return {"bytes": size * (rows * (dim + dim_v) + (sum(prefix) * groups if case["mass"] else 0)
                             + batch * heads * new * (dim + dim_v)),
            "flops": 2 * pairs * (dim + dim_v)}


def _exact_turn(x, positions, frequencies, interleaved, sign=1.0):
    """x ``[H, T, d]`` of one batch row as complex numbers times exp(i angle)."""
    half = frequencies.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       sign * torch.outer(positions.double(), frequencies))
    y = x.detach().double().clone()
    pairs = y[..., :2 * half].unflatten(-1, (half, 2) if interleaved else (2, half))
    pairs = pairs if interleaved else pairs.transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y[..., :2 * half] = (turned if interleaved else turned.transpose(-1, -2)).flatten(-2)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    batch, heads, groups, new = (case[n] for n in ("batch", "heads", "groups", "new"))
    if case["kind"] == "rotary":
        def turned(name, sign=1.0):
            return torch.stack([_exact_turn(x, s["positions"], s["frequencies"], case["interleaved"], sign) for x in s[name]])

        out = turned("q"), turned("k")
        return out + (turned("grad_q", -1.0), turned("grad_k", -1.0)) if case["train"] else out
    lens, page = _lengths(case), case["page"]
    table = s["table"].tolist()
    if case["kind"] == "append":
        step, counts = torch.arange(new, device="cuda"), _counts(case)
        q, k = (torch.stack([_exact_turn(s[n][b], case["first"] + lens[b] + step, s["frequencies"], case["interleaved"])
                             for b in range(batch)]) for n in "qk")
        pages = [s["k_pages"].double(), s["v_pages"].double()]
        for rows, x in zip(pages, (k, s["v"].double())):
            for b in range(batch):
                done = 0
                while done < counts[b]:
                    at = lens[b] + done
                    n = min(page - at % page, counts[b] - done)
                    rows[table[b][at // page], :, at % page:at % page + n] = x[b, :, done:done + n]
                    done += n
        return (q, k, *pages)
    per, share = heads // groups, batch // case["prefixes"]
    out = torch.zeros(batch, heads, new, case["dim_v"], dtype=torch.float64, device="cuda")
    hidden = torch.ones(new, new, dtype=torch.bool, device="cuda").triu(1)
    counts = s["prefix_lengths"].tolist()

    def held(pages, line, n, g):
        return pages[line[:-(-n // page)], g].flatten(0, 1)[:n].double() if n else pages.new_zeros((0, pages.size(-1))).double()

    for i, n in enumerate(counts):
        for g in range(groups):
            if s["prefix_table"] is not None:
                line = s["prefix_table"][i].tolist()
                kp, vp = held(s["k_pages"], line, n, g), held(s["v_pages"], line, n, g)
            else:
                kp, vp = s["prefix_k"][i, g, :n].double(), s["prefix_v"][i, g, :n].double()
            for b in range(i * share, (i + 1) * share):
                keys = torch.cat((kp, held(s["k_pages"], table[b], lens[b], g), s["k"][b, g].double()))
                vals = torch.cat((vp, held(s["v_pages"], table[b], lens[b], g), s["v"][b, g].double()))
                for h in range(g * per, (g + 1) * per):
                    logit = (s["q"][b, h].double() @ keys.T) * s["scale"]
                    if s["prefix_bias"] is not None:
                        logit[:, :n] += s["prefix_bias"][i, g, :n].double()
                    logit[:, n + lens[b]:][hidden] = -math.inf
                    out[b, h] = torch.softmax(logit, dim=-1) @ vals
    return out
