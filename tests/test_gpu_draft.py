"""Drafted tokens over the compressed cache: draft attention against the 64-bit attention of the packed rows, and the
cache after accept against one that was fed the accepted tokens."""

from __future__ import annotations

import pytest
import torch

from harness import STATE_FIELDS, to_np
from logkv_amd import LogKVStreamingAttention, LogStructuredKVCache, log_kv_draft_attention
from logkv_amd.log_kv_pack import pack_mid_kv, packed_dim, semantic_mid_attention_plan
from row_reference import check_close, reference, tree_mask
from workloads import Mixture, rope_tables

pytestmark = pytest.mark.gpu

B, G, HQ, N, R = 2, 2, 4, 512, 16


def new_engine(d, exact):
    cos, sin = rope_tables(N, d)
    cache = LogStructuredKVCache(
        (B, G, N, d), (B, G, N, d), B=8, recent_size=R, device="cuda", dtype=torch.bfloat16, semantic_clusters=True,
        cluster_k_max=4, semantic_s_h=16.0, semantic_flush_granularity=R, semantic_anchor_mode="mid",
        allocate_second_order=False, cos_cache=cos, sin_cache=sin, rope_n_elem=d, alpha_exact_tokens=8 if exact else 0,
        alpha_span_max_tokens=4, beta_novelty=exact, beta_adaptive_merge=exact)
    return LogKVStreamingAttention(cache, d ** -0.5, prefill_block=8)


def tokens(d, n, seed):
    mix = Mixture(B, G, d, clusters=4, seed=seed)
    q = torch.randn(B, HQ, n, d, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
    k, v, k_raw = mix.rows(n).cuda(), mix.rows(n).cuda(), mix.rows(n).cuda()
    return q, k, v, k_raw, mix.span_ends(0, n, 5)


def feed(engine, rows, a, b, exact):
    q, k, v, k_raw, ends = rows
    return engine(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], k_raw[:, :, a:b], input_pos=torch.arange(a, b, device="cuda"),
                  span_ends=[row[a:b] for row in ends] if exact else None)


def same_state(c1, c2):
    extra = ("alpha_k_raw", "alpha_v", "alpha_pos", "alpha_valid") if c1.alpha_exact_tokens else ()
    for f in STATE_FIELDS + extra:
        if hasattr(c1, f):
            assert (to_np(getattr(c1, f)) == to_np(getattr(c2, f))).all(), f
    n = c1.recent_count
    assert n == c2.recent_count and c1.token_count == c2.token_count
    for f in ("recent_k", "recent_v", "recent_k_raw"):
        assert torch.equal(getattr(c1, f)[:, :, :n], getattr(c2, f)[:, :, :n]), f
    assert torch.equal(c1.recent_pos[:, :n], c2.recent_pos[:, :n])


def draft_reference(engine, q, k, v, visible, scale):
    cache, pending = engine.cache, engine._log_kv_pending
    d = cache.k_dim
    pk, pv = (k[:, :, :1], v[:, :, :1]) if pending is None else pending[:2]
    ka, va = pack_mid_kv(cache, semantic_mid_attention_plan(cache), pk, pv, packed_dim(d, d))
    if pending is None:     # packed behind a row of its own, since there may be no other
        ka, va = ka[:, :, :-1], va[:, :, :-1]
    visible = visible.cpu().expand(B, *visible.shape[-2:])
    want, _, bound, _ = reference(q, k, v, ka[..., :d], va[..., :d], [ka.size(2)] * B, visible, scale, bias=ka[..., d].float())
    return want, bound


@pytest.mark.parametrize("prefill", [0, 1, 12, 37, 60])
@pytest.mark.parametrize("d,exact,T", [(64, True, 9), (128, False, 1), (64, False, 40)])
def test_draft_attends_the_packed_state_and_the_tree(d, exact, T, prefill):
    rows = tokens(d, prefill + T, 5 * prefill + T)
    engine = new_engine(d, exact)
    if prefill:
        feed(engine, rows, 0, prefill, exact)
    q, k, v, k_raw, ends = (x[:, :, prefill:] if isinstance(x, torch.Tensor) else [r[prefill:] for r in x] for x in rows)
    visible = torch.stack([tree_mask(T, s) for s in range(B)]).cuda()
    want, bound = draft_reference(engine, q, k, v, visible, engine.scale)
    out = engine.draft(q, k, v, k_raw, visible, input_pos=torch.arange(prefill, prefill + T, device="cuda"),
                       span_ends=ends if exact else None)
    check_close(out.view(B, T, HQ, d).transpose(1, 2), want, bound)
    # Again, over the packed prefix that the first left; and for one mask of all batch rows.
    again = engine.draft(q, k, v, k_raw, visible, span_ends=ends if exact else None)
    assert torch.equal(out, again)
    want, bound = draft_reference(engine, q, k, v, visible[:1], engine.scale)
    pending = engine._log_kv_pending
    one = log_kv_draft_attention(engine.cache, q.float(), k.float(), v.float(), visible[0], engine.scale,
                                 pending=None if pending is None else pending[:2])
    assert one.dtype == torch.float32
    check_close(one, want, bound)


@pytest.mark.parametrize("prefill", [7, 12, 29])
@pytest.mark.parametrize("path", [[0], [0, 1, 2], [1, 4, 5, 8], [0, 2, 3, 4, 6], [], [[0, 3, 5], [1, 2, 8]],
                                  list(range(20)), torch.tensor([[2, 3], [0, 19]])])
@pytest.mark.parametrize("exact", [True, False])
def test_accept_commits_what_a_call_would(prefill, path, exact):
    d, T = 64, 20
    rows = tokens(d, prefill + T + 6, 3)
    drafted, called = new_engine(d, exact), new_engine(d, exact)
    for e in (drafted, called):
        feed(e, rows, 0, prefill, exact)
    q, k, v, k_raw = (x[:, :, prefill:prefill + T] for x in rows[:4])
    ends = [r[prefill:prefill + T] for r in rows[4]] if exact else None
    pos = prefill + torch.arange(T, device="cuda") // 2
    drafted.draft(q, k, v, k_raw, tree_mask(T, 1).cuda(), input_pos=pos, span_ends=ends)
    drafted.accept(path)
    index = torch.as_tensor(path, dtype=torch.long)
    index = (index if index.dim() == 2 else index[None]).expand(B, -1).cuda()
    if index.size(1):
        pick = lambda x: torch.stack([x[b][:, index[b]] for b in range(B)])  # noqa: E731
        called(pick(q), pick(k), pick(v), pick(k_raw), input_pos=pos[index],
               span_ends=[[ends[b][i] for i in index[b].tolist()] for b in range(B)] if exact else None)
    assert (drafted._log_kv_pending is None) == (called._log_kv_pending is None)
    same_state(drafted.cache, called.cache)
    # The streams go on alike.
    for a, b in ((prefill + T, prefill + T + 1), (prefill + T + 1, prefill + T + 6)):
        assert torch.equal(feed(drafted, rows, a, b, exact), feed(called, rows, a, b, exact))
    same_state(drafted.cache, called.cache)


def test_a_draft_leaves_the_stream_as_it_was():
    d, prefill = 64, 37
    rows = tokens(d, prefill + 12, 17)
    plain, drafting = new_engine(d, True), new_engine(d, True)
    for e in (plain, drafting):
        feed(e, rows, 0, prefill, True)
    g = torch.Generator().manual_seed(2)
    for t in range(prefill, prefill + 12):
        x = [torch.randn(B, h, 5, d, generator=g).to(torch.bfloat16).cuda() for h in (HQ, G, G, G)]
        drafting.draft(*x, tree_mask(5, t).cuda(), span_ends=[[False] * 5] * B)
        assert torch.equal(feed(plain, rows, t, t + 1, True), feed(drafting, rows, t, t + 1, True)), t
    same_state(plain.cache, drafting.cache)
    with pytest.raises(RuntimeError, match="draft"):
        drafting.accept([0])


def test_drafts_behind_a_queued_flush_and_on_another_stream():
    """The cache's flushes on a stream of their own, the draft on a third: the same bits as on one stream."""
    d, prefill, T = 64, 30, 7
    rows = tokens(d, prefill + T, 23)
    one, streams = new_engine(d, False), new_engine(d, False)
    streams.cache.flush_stream = torch.cuda.Stream()
    x = [t[:, :, prefill:] for t in rows[:4]]
    visible = tree_mask(T, 3).cuda()
    for e in (one, streams):
        feed(e, rows, 0, prefill, False)
    want = one.draft(*x, visible)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = streams.draft(*x, visible)
        streams.accept([0, 1, 3])
    side.synchronize()
    one.accept([0, 1, 3])
    assert torch.equal(want, got)
    same_state(one.cache, streams.cache)


def test_refusals():
    d, T = 64, 4
    engine = new_engine(d, True)
    q, k, v, k_raw, ends = tokens(d, T, 1)
    visible = tree_mask(T, 1).cuda()
    with pytest.raises(ValueError, match="span"):
        engine.draft(q, k, v, k_raw, visible)
    with pytest.raises(ValueError, match="visible"):
        engine.draft(q, k, v, k_raw, visible[:3, :3], span_ends=ends)
    with pytest.raises(ValueError, match="visible"):
        engine.draft(q, k, v, k_raw, visible.float(), span_ends=ends)
    with pytest.raises(ValueError, match="k_raw"):
        engine.draft(q, k, v, k_raw[:, :, :2], visible, span_ends=ends)
    with pytest.raises(ValueError):
        engine.draft(q, k[:1], v[:1], k_raw[:1], visible, span_ends=ends)
    with pytest.raises(ValueError, match="pending"):
        log_kv_draft_attention(engine.cache, q, k, v, visible, engine.scale, pending=(k, v))
    with pytest.raises(NotImplementedError, match="gradient"):
        log_kv_draft_attention(engine.cache, q.float().requires_grad_(), k, v, visible, engine.scale)
    with pytest.raises(RuntimeError, match="draft"):
        engine.accept([0])
    engine.draft(q, k, v, k_raw, visible, span_ends=ends)
    for path in ([4], [-1], [1, 0], [2, 2], [[0], [1], [2]], [[0], [1, 2]]):
        with pytest.raises(ValueError, match="path"):
            engine.accept(path)
    engine.accept([0, 3])
    assert engine.cache.token_count == 2
