"""Rows hidden by a large finite bias, of the sizes at which float32 no longer holds the fp16 probabilities' scale beside
the logits: they weigh nothing beside others, and alone they leave a mean of their values."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import log_kv_tree_attention
from row_lanes import check_lane, lane
from row_reference import tree_mask
from test_gpu_row_attention import inputs

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
MASKS = [-1e4, -1.2e7, -1.5e7, -2e7, -3e7, -5e7, -1e8, -1.8e8, -3e8, -1e9, -1e30]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rep,T,d", [(2, 5, 64), (2, 13, 128), (2, 9, 256), (2, 20, 64), (3, 40, 128), (4, 50, 64)])
def test_rows_hidden_by_a_large_bias(rep, T, d, dtype):
    cap = 400
    q, k, v, ck, cv = inputs(1, 1, rep, T, cap, d, d, dtype, 30)
    see = tree_mask(T, 3)
    for mask in MASKS:
        bias = torch.zeros(1, 1, cap, device="cuda")
        bias[:, :, :130] = mask      # whole tiles, met first
        bias[:, :, 300:333] = mask
        out = log_kv_tree_attention(q, k, v, ck, cv, cap, see.cuda(), d ** -0.5, bias=bias)
        want, bound, _, _ = lane(q, k, v, ck, cv, 0, 0, cap, see, d ** -0.5, bias)
        check_lane(out[0], want, bound, f"bias {mask}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rep,T,d", [(2, 5, 64), (2, 20, 64), (3, 40, 128), (4, 50, 64)])
def test_only_rows_of_a_large_bias(rep, T, d, dtype):
    """No other row to see: the logits are what float32 leaves of them beside the bias, the output a mean of values."""
    cap = 400
    q, k, v, ck, cv = inputs(1, 1, rep, T, cap, d, d, dtype, 31)
    none = torch.zeros(T, T, dtype=torch.bool, device="cuda")
    lo, hi = cv[0, 0].float().amin(0), cv[0, 0].float().amax(0)
    slack = 2.0 ** -7 * torch.maximum(lo.abs(), hi.abs())
    for mask in MASKS + [5e7, 1e8]:
        bias = torch.full((1, 1, cap), mask, device="cuda")
        out = log_kv_tree_attention(q, k, v, ck, cv, cap, none, d ** -0.5, bias=bias).float()
        assert bool(torch.isfinite(out).all()), mask
        assert bool(((out >= lo - slack) & (out <= hi + slack)).all()), mask


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rep,T", [(2, 5), (2, 20), (3, 40), (4, 50)])
def test_very_large_logits(rep, T, dtype):
    """One row's logit stands millions above the others': the output is its value."""
    d, cap = 64, 300
    _, k, v, ck, cv = inputs(1, 1, rep, T, cap, d, d, dtype, 33)
    for size in (300.0, 1000.0, 1500.0, 2000.0):
        q = torch.full((1, rep, T, d), size, dtype=dtype, device="cuda")
        keys = torch.full((1, 1, cap, d), size / 2, dtype=dtype, device="cuda")
        keys[:, :, 100] = size
        keys[:, :, 200] = size * 0.875
        out = log_kv_tree_attention(q, k, v, keys, cv, cap, torch.zeros(T, T, dtype=torch.bool, device="cuda"), 0.125)
        want = cv[0, 0, 100].double().expand(rep, T, d)
        check_lane(out[0], want, 2.0 ** -10 * want.abs(), f"size {size}")
