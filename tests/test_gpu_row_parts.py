"""bf16 probabilities enter the value products as two rounded parts, so that their sums have no bias against the divisor."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import log_kv_tree_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("rep,T", [(2, 8), (2, 13), (2, 20), (3, 40), (4, 50)])
def test_parts_are_rounded(rep, T, d):
    """Two rows of values 1 and -1 and nearly equal logits: the larger probability is 1 before the division, the smaller
    one, just below it, is held in parts. Rounded, they err either way: by at most 2^-17 of a half of the weight and the
    output's 2^-8 of 2^-10, with no mean but the exponentials' 2^-22 and what 2048 queries or more leave of those
    (five deviations: 2^-22). Cut, they would all err to one side, by 2^-18 in the mean."""
    B, G, scale = 16, 8, 0.7
    q = torch.zeros(B, G * rep, T, d)
    q[..., 0] = torch.rand(B, G * rep, T, generator=torch.Generator().manual_seed(rep * T + d)) * 2 - 1
    ck, cv = torch.zeros(B, G, 2, d), torch.ones(B, G, 2, d)
    ck[:, :, 1, 0], cv[:, :, 1] = 2.0 ** -9, -1.0
    q, ck, cv = (x.to(torch.bfloat16).cuda() for x in (q, ck, cv))
    own = torch.zeros(B, G, T, d, dtype=torch.bfloat16, device="cuda")
    out = log_kv_tree_attention(q, own, own, ck, cv, 2, torch.zeros(T, T, dtype=torch.bool, device="cuda"), scale)
    s = q[..., 0].double() * 2.0 ** -9 * scale
    want = -torch.tanh(s / 2)
    err = out.double()[..., 0] - want
    assert torch.equal(out, out[..., :1].expand_as(out))
    assert float(err.abs().max()) <= 2.0 ** -18 + 2.0 ** -18 + 2.0 ** -20
    assert abs(float((err * torch.sign(s)).mean())) <= 2.0 ** -20
