"""A draft's logits are the ones that a call computes: slots' log-mass times ``scale * bf16(1 / scale)``."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import LogKVStreamingAttention, LogStructuredKVCache, log_kv_chunk_attention
from logkv_amd.log_kv_pack import pack_mid_kv, packed_dim, semantic_mid_attention_plan
from row_lanes import check_lane, lane
from workloads import Mixture, rope_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 8, 20, 50])
@pytest.mark.parametrize("d,scale", [(96, None), (64, 0.0995), (128, 0.0995)])
def test_a_drafted_chain_is_a_calls_chunk(d, scale, T):
    B, G, HQ, N, R, n = 2, 2, 4, 2048, 32, 1536
    scale = scale or d ** -0.5
    factor = scale * float(torch.tensor(1.0 / scale).to(torch.bfloat16))
    cos, sin = rope_tables(N, d)
    cache = LogStructuredKVCache(
        (B, G, N, d), (B, G, N, d), B=4, recent_size=R, device="cuda", dtype=torch.bfloat16, semantic_clusters=True,
        cluster_k_max=2, semantic_s_h=16.0, semantic_flush_granularity=R, semantic_anchor_mode="mid",
        allocate_second_order=False, cos_cache=cos, sin_cache=sin, rope_n_elem=d)
    engine = LogKVStreamingAttention(cache, scale, prefill_block=32)
    mix = Mixture(B, G, d, clusters=2, seed=4)
    q = torch.randn(B, HQ, n + T, d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    k, v, k_raw = (mix.rows(n + T).cuda() for _ in range(3))
    engine(q[:, :, :n], k[:, :, :n], v[:, :, :n], k_raw[:, :, :n], input_pos=torch.arange(n, device="cuda"))
    q, k, v, k_raw = (x[:, :, n:] for x in (q, k, v, k_raw))
    causal = torch.ones(T, T, dtype=torch.bool).tril()
    called = log_kv_chunk_attention(cache, q, k, v, scale, 0.0)
    drafted = engine.draft(q, k, v, k_raw, causal.cuda()).view(B, T, HQ, d).transpose(1, 2)
    ka, va = pack_mid_kv(cache, semantic_mid_attention_plan(cache), k, v, packed_dim(d, d))
    rows = ka.size(2) - T
    mass = ka[..., d].float()
    # A logit that is off by (factor - 1) log w would be off by more than the bound allows.
    assert float((mass * (factor - 1)).abs().max()) > 0.002
    for b in range(B):
        for g in range(G):
            want, bound, _, _ = lane(q, k, v, ka[:, :, :rows, :d], va[:, :, :rows, :d], b, g, rows, causal, scale, mass * factor)
            heads = slice(g * HQ // G, (g + 1) * HQ // G)
            check_lane(drafted[b, heads], want, bound, "draft")
            # The call's own kernels hold a probability to 2^-11.
            check_lane(called[b, heads], want, bound + 2.0 ** -10 * want.abs().amax(-1, keepdim=True) + 2.0 ** -11, "call")
