"""A PagedKVCache as it is used: prompts, steps, drafts, shared prefixes in its pages and compressed documents, against
one causal attention over everything in 64 bits; and the rotation in front of training attention."""

from __future__ import annotations

import pytest
import torch

from harness import to_np  # noqa: F401
from logkv_amd import (LogKVStreamingAttention, LogStructuredKVCache, PagedKVCache, log_kv_rotary, rotary_frequencies,
                       rotary_tables)
from logkv_amd.log_kv_pack import pack_mid_kv, packed_dim, semantic_mid_attention_plan
from paged_reference import rotate, within
from row_reference import check_close, reference, tree_mask
from workloads import Mixture

pytestmark = pytest.mark.gpu


def make(B, H, T, d, dtype, seed, factor=1.0):
    return (factor * torch.randn(B, H, T, d, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def rows(B, H, G, T, dk, dv, dtype, seed):
    return make(B, H, T, dk, dtype, seed, 2.0), make(B, G, T, dk, dtype, seed + 1), make(B, G, T, dv, dtype, seed + 2)


def causal(B, T):
    return torch.ones(T, T, dtype=torch.bool).tril().expand(B, T, T)


class Mirror:
    """What a cache should hold: each sequence's rotated keys (as the pages' dtype has them) and values."""

    def __init__(self, B, G, dk, dv, dtype, frequencies, interleaved=False, amplitude=1.0):
        self.dtype, self.f, self.interleaved, self.amplitude = dtype, frequencies, interleaved, amplitude
        self.k = [torch.zeros(G, 0, dk, dtype=dtype) for _ in range(B)]
        self.v = [torch.zeros(G, 0, dv, dtype=dtype) for _ in range(B)]

    def turned(self, x, pos, to):
        """As the library rounds it (its rotation is tested on its own)."""
        if self.f is None:
            return x.to(to)
        y, _ = log_kv_rotary(x, None, self.f, pos.cuda(), interleaved=self.interleaved, amplitude=self.amplitude)
        return y.to(to)

    def step(self, q, k, v, first, counts=None, visible=None, store=True, positions=None, scale=None):
        """(attention, bound) of new tokens, which are then held."""
        B, T = q.size(0), q.size(2)
        pos = positions if positions is not None else torch.stack(
            [first[b] + self.k[b].size(1) + torch.arange(T) for b in range(B)])
        q2, k2, v2 = self.turned(q, pos, self.dtype), self.turned(k, pos, self.dtype), v.to(self.dtype)
        n = [x.size(1) for x in self.k]
        cap = max(max(n), 1)
        ck, cv = (torch.zeros(B, x[0].size(0), cap, x[0].size(2), dtype=self.dtype) for x in (self.k, self.v))
        for b in range(B):
            ck[b, :, :n[b]], cv[b, :, :n[b]] = self.k[b], self.v[b]
        out, _, bound, _ = reference(q2, k2, v2, ck, cv, n, causal(B, T) if visible is None else visible.cpu().expand(B, T, T),
                                     scale, counts=counts)
        if store:
            for b in range(B):
                live = T if counts is None else int(counts[b])
                self.k[b] = torch.cat((self.k[b], k2[b, :, :live].cpu()), dim=1)
                self.v[b] = torch.cat((self.v[b], v2[b, :, :live].cpu()), dim=1)
        return out, bound


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("dk,dv,rotated,interleaved,prefixes", [(64, 64, 64, False, 0), (128, 64, 32, True, 2),
                                                                (192, 128, 64, False, 1), (64, 64, 0, False, 4)])
def test_prompts_steps_and_drafts(dk, dv, rotated, interleaved, prefixes, dtype):
    B, H, G, page = 4, 4, 2, 16
    f = rotary_frequencies(rotated, scaling=dict(kind="linear", factor=4.0))[0] if rotated else None
    cache = PagedKVCache(B, G, dk, dv, 60, scale=dk ** -0.5, max_rows=120, page_size=page, frequencies=f,
                         interleaved=interleaved, amplitude=1.25 if rotated else 1.0, dtype=dtype)
    scale = cache.scale
    kw = dict(frequencies=f, interleaved=interleaved, amplitude=cache.amplitude)
    # Prefixes, in two blocks.
    done, first = Mirror(max(prefixes, 1), G, dk, dv, dtype, **kw), [0] * B
    if prefixes:
        for T, seed in ((37, 1), (8, 5)):
            q, k, v = rows(prefixes, H, G, T, dk, dv, dtype, seed)
            want, bound = done.step(q, k, v, [0] * prefixes, scale=scale)
            check_close(cache.prefix(q, k, v), want, bound, "prefix")
    mirror = Mirror(B, G, dk, dv, dtype, **kw)
    if prefixes:     # a sequence's rows follow its prefix's
        run = B // prefixes
        mirror.k, mirror.v = ([x[b // run] for b in range(B)] for x in (done.k, done.v))
    for round_ in range(2):
        # A padded prompt, steps of one and of several tokens, a draft between.
        for T, seed, counts in ((21, 10, [21, 0, 7, 16]), (1, 20, None), (5, 30, [5, 5, 1, 0]), (1, 40, None)):
            q, k, v = rows(B, H, G, T, dk, dv, dtype, seed + round_)
            see = tree_mask(T, seed).cuda()
            depth = torch.stack([torch.as_tensor(mirror.k[b].size(1) + torch.arange(T)) for b in range(B)])
            want, bound = mirror.step(q, k, v, first, visible=see, store=False, positions=depth, scale=scale)
            check_close(cache.draft(q, k, v, see, positions=None if f is None else depth.cuda()), want, bound, "draft")
            want, bound = mirror.step(q, k, v, first, counts=counts, scale=scale)
            given = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
            check_close(cache(q, k, v, counts=given), want, bound, ("call", round_, T))
        assert cache.lengths.tolist() == [x.size(1) - (done.k[0].size(1) if prefixes else 0) for x in mirror.k]
        held = cache.free_pages
        cache.trim()
        need = sum(-(-n // page) for n in cache.lengths.tolist()) + prefixes * -(-cache._prefix_rows // page)
        assert cache.free_pages == 60 - need >= held
        if round_ == 0:    # two sequences end, their pages serve others
            cache.free([0, 2])
            for b in (0, 2):
                p = done.k[0].size(1) if prefixes else 0
                mirror.k[b], mirror.v[b] = mirror.k[b][:, :p], mirror.v[b][:, :p]
    cache.reset()
    assert cache.free_pages == 60 and cache.lengths.tolist() == [0] * B
    q, k, v = rows(B, H, G, 2, dk, dv, dtype, 77)
    want, bound = Mirror(B, G, dk, dv, dtype, **kw).step(q, k, v, [0] * B, scale=scale)
    check_close(cache(q, k, v), want, bound, "after reset")


def test_activations_of_another_dtype():
    B, H, G, d = 2, 2, 1, 64
    f = rotary_frequencies(d)[0]
    cache = PagedKVCache(B, G, d, d, 8, scale=0.125, max_rows=32, page_size=16, frequencies=f)
    mirror = Mirror(B, G, d, d, torch.bfloat16, f)
    for T, seed in ((9, 1), (1, 4)):
        q, k, v = rows(B, H, G, T, d, d, torch.float32, seed)
        want, bound = mirror.step(q, k, v, [0] * B, scale=0.125)
        out = cache(q, k, v)
        assert out.dtype == torch.float32
        check_close(out, want, bound)


def new_engine(batch, d, exact, recent=16, n=512):
    f = rotary_frequencies(d)[0]
    cos, sin = rotary_tables(f, n)
    cache = LogStructuredKVCache(
        (batch, 2, n, d), (batch, 2, n, d), B=8, recent_size=recent, device="cuda", dtype=torch.bfloat16, semantic_clusters=True,
        cluster_k_max=4, semantic_s_h=16.0, semantic_flush_granularity=recent, semantic_anchor_mode="mid",
        allocate_second_order=False, cos_cache=cos, sin_cache=sin, rope_n_elem=d, alpha_exact_tokens=8 if exact else 0,
        alpha_span_max_tokens=4, beta_novelty=exact, beta_adaptive_merge=exact)
    return LogKVStreamingAttention(cache, d ** -0.5, prefill_block=8), f


@pytest.mark.parametrize("documents,exact,tokens", [(1, False, 60), (2, True, 37), (1, True, 0), (4, False, 5)])
def test_answers_behind_compressed_documents(documents, exact, tokens):
    """The documents are rotated, compressed and streamed by LogKV; the answers' rows stand in pages behind them."""
    d, G, H, B = 64, 2, 4, 4
    engine, f = new_engine(documents, d, exact)
    mix = Mixture(documents, G, d, clusters=4, seed=3)
    if tokens:
        k_raw, v = mix.rows(tokens).cuda(), mix.rows(tokens).cuda()
        q = make(documents, H, tokens, d, torch.bfloat16, 5)
        pos = torch.arange(tokens, device="cuda")
        q2, k = log_kv_rotary(q, k_raw, f, pos)
        ends = mix.span_ends(0, tokens, 5) if exact else None
        engine(q2, k, v, k_raw, input_pos=pos, span_ends=ends)
    cache = PagedKVCache(B, G, d, d, 40, scale=engine.scale, max_rows=100, page_size=16, frequencies=f)
    cache.share(engine)
    run = B // documents
    # The document's rows as LogKV packs them.
    pending = engine._log_kv_pending
    pk, pv = (make(documents, G, 1, d, torch.bfloat16, 8),) * 2 if pending is None else pending[:2]
    ka, va = pack_mid_kv(engine.cache, semantic_mid_attention_plan(engine.cache), pk, pv, packed_dim(d, d))
    if pending is None:
        ka, va = ka[:, :, :-1], va[:, :, :-1]
    P = ka.size(2)
    mirror = Mirror(B, G, d, d, torch.bfloat16, f)
    mirror.k, mirror.v = ([x[b // run, :, :, :d].cpu() for b in range(B)] for x in (ka, va))
    bias = torch.stack([ka[b // run, :, :, d].float().cpu() for b in range(B)])
    for T, seed, counts in ((13, 1, [13, 4, 0, 9]), (1, 5, None), (3, 9, None)):
        q, k, v = rows(B, H, G, T, d, d, torch.bfloat16, seed)
        n = [x.size(1) for x in mirror.k]
        pos = torch.stack([tokens + n[b] - P + torch.arange(T) for b in range(B)])
        q2, k2 = mirror.turned(q, pos, q.dtype), mirror.turned(k, pos, k.dtype)
        ck, cv = (torch.zeros(B, G, max(n) + 1, d, dtype=torch.bfloat16) for _ in range(2))
        add = torch.zeros(B, G, max(n) + 1)
        for b in range(B):
            ck[b, :, :n[b]], cv[b, :, :n[b]], add[b, :, :P] = mirror.k[b], mirror.v[b], bias[b]
        want, _, bound, _ = reference(q2, k2, v, ck, cv, n, causal(B, T), engine.scale, bias=add, counts=counts)
        given = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
        drafted = cache.draft(q, k, v, causal(1, T)[0].cuda(), positions=pos.cuda())
        out = cache(q, k, v, counts=given)
        check_close(out, want, bound, T)
        if counts is None:
            assert torch.equal(drafted, out)
        for b in range(B):
            live = T if counts is None else counts[b]
            mirror.k[b] = torch.cat((mirror.k[b], k2[b, :, :live].cpu()), dim=1)
            mirror.v[b] = torch.cat((mirror.v[b], v[b, :, :live].cpu()), dim=1)


def test_documents_that_do_not_fit():
    engine, _ = new_engine(2, 64, False)
    for cache in (PagedKVCache(3, 2, 64, 64, 4, scale=0.125, max_rows=16), PagedKVCache(4, 1, 64, 64, 4, scale=0.125, max_rows=16),
                  PagedKVCache(4, 2, 128, 64, 4, scale=0.125, max_rows=16),
                  PagedKVCache(4, 2, 64, 64, 4, scale=0.125, max_rows=16, dtype=torch.float16)):
        with pytest.raises(ValueError):
            cache.share(engine)
    cache = PagedKVCache(4, 2, 64, 64, 4, scale=0.125, max_rows=16)
    cache.share(engine.cache)
    with pytest.raises(RuntimeError):
        cache.prefix(*rows(2, 4, 2, 3, 64, 64, torch.bfloat16, 1))


def test_captures_are_refused():
    cache = PagedKVCache(2, 1, 64, 64, 4, scale=0.125, max_rows=16)
    q, k, v = rows(2, 2, 1, 1, 64, 64, torch.bfloat16, 1)
    cache(q, k, v)
    before = cache.lengths.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            cache(q, k, v)
        q.add_(0)
    torch.cuda.synchronize()
    assert torch.equal(cache.lengths, before) and cache._bound == [1, 1]


def test_prefix_attention_in_a_graph():
    """Over a compressed document that nobody has read yet: the capture, which runs nothing, leaves nothing behind; replays
    between the program's own calls equal them."""
    from logkv_amd import log_kv_prefix_attention

    engine, _ = new_engine(2, 64, False)
    q, k, v = rows(2, 4, 2, 150, 64, 64, torch.bfloat16, 5)
    engine(q, k, v, k, input_pos=torch.arange(150, device="cuda"), span_ends=None)
    cache = engine.cache
    pending = None if engine._log_kv_pending is None else engine._log_kv_pending[:2]
    q, k, v = rows(4, 4, 2, 1, 64, 64, torch.bfloat16, 9)
    pages = make(4, 2, 16, 64, torch.bfloat16, 12), make(4, 2, 16, 64, torch.bfloat16, 13)
    table = torch.arange(4, dtype=torch.int32, device="cuda")[:, None].contiguous()
    n = torch.tensor([3, 0, 16, 7], dtype=torch.int32, device="cuda")

    def call():
        with torch.no_grad():
            return log_kv_prefix_attention(cache, q, k, v, *pages, table, n, 0.125, pending=pending)

    cache._mid_decode_state = None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    assert cache._mid_decode_state is None
    first = call()      # packs for itself
    for i in range(3):
        q.normal_(generator=torch.Generator("cuda").manual_seed(i))
        n.add_(1).clamp_(max=16)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and not torch.equal(got, first)


def test_compression_accounting():
    from types import SimpleNamespace as S

    from logkv_amd import cache_compression_snapshot

    cache = PagedKVCache(4, 2, 64, 64, 12, scale=0.125, max_rows=32, page_size=16)
    cache.prefix(*rows(2, 4, 2, 20, 64, 64, torch.bfloat16, 1))
    cache(*rows(4, 4, 2, 3, 64, 64, torch.bfloat16, 4))
    model = S(transformer=S(h=[S(attn=S(kv_cache=cache))]))
    counts = cache_compression_snapshot(model, 23)
    assert counts["retained_slots"] == (2 * 20 + 4 * 3) * 2 and counts["dense_slots"] == 23 * 8


def test_rotation_in_front_of_training_attention():
    """Gradients of a rotated, streamed training step: those of the attention, rotated back."""
    from logkv_amd import LogKVStreamTrainingAttention

    d, T, H, G = 64, 48, 4, 2
    f = rotary_frequencies(d)[0]
    mix = Mixture(1, G, d, clusters=4, seed=11)
    k_raw, v = mix.rows(T).cuda(), mix.rows(T).cuda()
    q_raw, dout = make(1, H, T, d, torch.bfloat16, 1), make(1, H, T, d, torch.bfloat16, 2)
    pos = torch.arange(T, device="cuda")

    def cache():
        engine, _ = new_engine(1, d, False)
        c = engine.cache
        c.semantic_replay_updates = True
        return c

    a, b = q_raw.clone().requires_grad_(), k_raw.clone().requires_grad_()
    q, k = log_kv_rotary(a, b, f, pos)
    y = LogKVStreamTrainingAttention.apply(q, k, v, cache(), d ** -0.5, 16, 0.0, k_raw, None)
    da, db = torch.autograd.grad(y, (a, b), dout)
    # The attention's own gradients, of rows that are leaves.
    q1, k1 = q.detach().requires_grad_(), k.detach().requires_grad_()
    y1 = LogKVStreamTrainingAttention.apply(q1, k1, v, cache(), d ** -0.5, 16, 0.0, k_raw, None)
    assert torch.equal(y, y1)
    dq, dk = torch.autograd.grad(y1, (q1, k1), dout)
    at = pos.cpu().expand(1, -1)
    within(da, *rotate(dq, f, at, sign=-1.0))
    within(db, *rotate(dk, f, at, sign=-1.0))
