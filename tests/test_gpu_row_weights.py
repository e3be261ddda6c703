"""Weights of weight attention in every form of its passes, and where a key holds an infinity (row_lanes.py derives the
bounds)."""

from __future__ import annotations

import math

import pytest
import torch

from logkv_amd import log_kv_weight_attention
from row_lanes import check_lane, check_weights, lane
from test_gpu_row_attention import inputs

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def run(q, k, v, ck, cv, lengths, lanes, counts=None, seed=8):
    B, G, cap, d = ck.shape
    rep, T = q.size(1) // G, q.size(2)
    w = torch.rand(B, G, cap, generator=torch.Generator().manual_seed(seed)).cuda()
    before, old_k, old_v, scale = w.clone(), ck.clone(), cv.clone(), d ** -0.5
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    c = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = log_kv_weight_attention(q, k, v, ck, cv, w, n, scale, counts=c)
    see = torch.ones(T, T, dtype=torch.bool).tril()
    for b, g in lanes:
        live = T if counts is None else counts[b]
        want, bound, column, rel = lane(q, k, v, old_k, old_v, b, g, lengths[b], see, scale, live=live)
        check_lane(out[b, g * rep:(g + 1) * rep], want, bound, f"lane {b}, {g}")
        check_weights(w[b, g], before[b, g], column[:lengths[b] + live], lengths[b], cap, rel, rep * T, f"lane {b}, {g}")
    return out, w


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,G,rep,T,cap", [
    (1, 2, 2, 100, 1200),       # two waves to 32 keys, each half of the queries
    (2, 8, 2, 70, 5000),        # 32 keys a wave
    (2, 8, 2, 100, 9000),       # 64 keys a wave
])
def test_forms_of_the_weight_pass(B, G, rep, T, cap, d, dtype):
    lengths = [cap - T - 37 * b for b in range(B)]
    q, k, v, ck, cv = inputs(B, G, rep, T, cap, d, d, dtype, T + d)
    run(q, k, v, ck, cv, lengths, [(0, 0), (B - 1, G - 1)])


@pytest.mark.parametrize("T", [1, 3])
def test_four_columns_a_thread(T):
    """Few queries over lanes of many rows: the weights' pass takes four columns a thread."""
    B, G, cap = 4, 8, 33000
    q, k, v, ck, cv = inputs(B, G, 2, T, cap, 64, 64, BF16, 40 + T)
    run(q, k, v, ck, cv, [cap - T, 20001, 31, 0], [(0, 0), (1, 7), (2, 3), (3, 0)])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rep,T,count,d", [(2, 5, 5, 64), (2, 33, 33, 64), (2, 32, 32, 64), (2, 40, 39, 128), (1, 100, 1, 128),
                                           (3, 50, 17, 64), (1, 45, 45, 256)])
def test_keys_of_minus_infinite_logits_weigh_nothing(rep, T, count, d, dtype):
    """Keys with an infinity that gives every query a logit of -inf, in the cache and among the new rows: weight 0, also
    where the queries do not fill their last tile or the batch is padded."""
    q, k, v, ck, cv = inputs(2, 1, rep, T, 200, d, d, dtype, 3 * T + d)
    q[..., 0] = q[..., 0].abs() + 0.5
    ck[:, :, 5, 0] = ck[:, :, 64, 0] = -math.inf
    counts = [count, T]
    if count > 2:
        k[:, :, 1, 0] = -math.inf
    for b, c in enumerate(counts):   # padding holds anything
        q[b, :, c:], k[b, :, c:] = math.nan, math.nan
    q0 = q.clone()
    q0[torch.isnan(q0)] = 0.0        # for the 64-bit form, which masks them
    k0 = torch.where(torch.isnan(k), torch.zeros_like(k), k)
    w = torch.zeros(2, 1, 200, device="cuda")
    old_k, old_v, lengths = ck.clone(), cv.clone(), [100, 65]
    out = log_kv_weight_attention(q, k, v, ck, cv, w, torch.tensor(lengths, dtype=torch.int32, device="cuda"), d ** -0.5,
                                  counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
    see = torch.ones(T, T, dtype=torch.bool).tril()
    for b, n in enumerate(lengths):
        want, bound, column, rel = lane(q0, k0, v, old_k, old_v, b, 0, n, see, d ** -0.5, live=counts[b])
        check_lane(out[b], want, bound)
        assert float(column[5]) == 0.0 and float(w[b, 0, 5]) == 0.0 and float(w[b, 0, 64]) == 0.0
        check_weights(w[b, 0], torch.zeros(200, device="cuda"), column[:n + counts[b]], n, 200, rel, rep * T)
