"""What the number of bits in a probability or a value decides: outputs that cancel, values that are small beside others
(row_lanes.py derives the bounds)."""

from __future__ import annotations

import math

import pytest
import torch

from logkv_amd import log_kv_tree_attention
from row_lanes import check_lane, lane
from test_gpu_row_attention import inputs

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
# Queries of a KV group: one and two blocks of 16 in the streaming kernel, the tiled kernel's blocks of 64, 128 and 256.
QUERIES = [(2, 8), (2, 13), (2, 20), (3, 40), (4, 50)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rep,T", QUERIES)
def test_two_rows_of_opposite_values(rep, T, d, dtype):
    """Two rows share nearly all of the weight and hold opposite values: the output is the difference of two probabilities
    near a half, and shows the rounding of each."""
    g = torch.Generator().manual_seed(rep * T + d)
    q = torch.zeros(1, rep, T, d)
    q[..., 0] = torch.rand(rep, T, generator=g) * 2 - 1      # the logits' difference, times 0.7 2^-9
    q[..., 1] = 4.0
    ck = torch.zeros(1, 1, 90, d)
    ck[:, :, :, 1] = -20.0                                   # all others: e^-56
    ck[:, :, 10, 1] = ck[:, :, 77, 1] = 0.0
    ck[:, :, 77, 0] = 2.0 ** -9
    cv = torch.randn(1, 1, 90, d, generator=g)
    cv[:, :, 77] = -cv[:, :, 10]
    q, ck, cv = (x.to(dtype).cuda() for x in (q, ck, cv))
    k, v = torch.zeros(1, 1, T, d, dtype=dtype, device="cuda"), torch.zeros(1, 1, T, d, dtype=dtype, device="cuda")
    see = torch.zeros(T, T, dtype=torch.bool)
    out = log_kv_tree_attention(q, k, v, ck, cv, 90, see.cuda(), 0.7)
    want, bound, _, _ = lane(q, k, v, ck, cv, 0, 0, 90, see, 0.7)
    assert float(want.abs().max()) < 2.0 ** -10 * float(cv.abs().max())
    check_lane(out[0], want, bound)


@pytest.mark.parametrize("where", ["feature", "rows", "hidden"])
@pytest.mark.parametrize("rep,T", QUERIES)
def test_small_values_beside_ordinary_ones(rep, T, where):
    """bf16 values far below 2^-17 keep their relative accuracy whatever stands beside them: a small feature, queries
    whose weight lies on small rows, a hidden row of ordinary size."""
    d, cap = 64, 200
    q, k, v, ck, cv = inputs(1, 1, rep, T, cap, d, d, torch.float32, 25)
    bias = torch.zeros(1, 1, cap, device="cuda")
    if where == "feature":
        cv[..., 5], v[..., 5] = cv[..., 5] * 1e-7, v[..., 5] * 1e-7
    else:
        cv[:, :, 1:], v = cv[:, :, 1:] * 1e-9, v * 1e-9
        bias[:, :, 0] = -math.inf if where == "hidden" else -200.0     # e^-200 of the row's ordinary values
    q, k, v, ck, cv = (x.to(BF16) for x in (q, k, v, ck, cv))
    see = torch.eye(T, dtype=torch.bool)
    out = log_kv_tree_attention(q, k, v, ck, cv, cap, see.cuda(), d ** -0.5, bias=bias)
    want, bound, _, _ = lane(q, k, v, ck, cv, 0, 0, cap, see, d ** -0.5, bias)
    check_lane(out[0], want, bound)
    if where != "feature":
        assert bool((out != 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("queries", [20, 32])
def test_small_values_of_17_to_32_queries_over_many_rows(queries, dtype):
    d, cap, n = 128, 131100, 3000
    q, k, v, ck, cv = inputs(1, 1, 1, queries, cap, d, d, dtype, 26)
    small = 1e-7 if dtype == BF16 else 1e-2
    cv[..., 7], v[..., 7] = cv[..., 7] * small, v[..., 7] * small
    see = torch.eye(queries, dtype=torch.bool)
    out = log_kv_tree_attention(q, k, v, ck, cv, n, see.cuda(), d ** -0.5)
    want, bound, _, _ = lane(q, k, v, ck, cv, 0, 0, n, see, d ** -0.5)
    check_lane(out[0], want, bound)
