"""Tiled row attention over shares of several tiles (row_reference.py derives the bounds): every block form, with and
without a bias, trees and causal chunks. Sizes are such that a share holds four 64-row tiles or more: the blocks of all
lanes come near the CUs, so that the rows are split into few shares."""

from __future__ import annotations

import pytest
import torch

from logkv_amd import log_kv_tree_attention, log_kv_weight_attention
from row_reference import check_close, reference, tree_mask
from test_gpu_row_attention import inputs

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def check_token(out, q, k, v, ck, cv, lane, n, t, see, scale, bias=None):
    """The output of token t of (batch row, KV head) ``lane`` over n rows and the own rows ``see``."""
    (b, g), rep = lane, q.size(1) // k.size(1)
    heads = slice(g * rep, (g + 1) * rep)
    keys = torch.cat((ck[b, g, :n], k[b, g, see]))[None, None]
    vals = torch.cat((cv[b, g, :n], v[b, g, see]))[None, None]
    add = None
    if bias is not None:
        add = torch.cat((bias[b, g, :n].float(), torch.zeros(len(see) - 1, device="cuda")))[None, None]
    want, _, bound, _ = reference(q[b:b + 1, heads, t:t + 1], keys[:, :, -1:], vals[:, :, -1:], keys[:, :, :-1], vals[:, :, :-1],
                                  [keys.size(2) - 1], torch.ones(1, 1, 1, dtype=torch.bool), scale, bias=add)
    check_close(out[b:b + 1, heads, t:t + 1], want, bound, f"lane {lane}, token {t}")


FORMS = [
    # B, G, rep, T, rows, d: queries of a KV group (a block holds 64, 128 or 256), tiles of a share
    (16, 8, 2, 20, 1500, 64),     # 40, 9
    (8, 8, 2, 26, 1500, 128),     # 52, 5
    (8, 4, 4, 30, 1500, 64),      # 120, 5
    (8, 8, 4, 30, 1100, 128),     # 120, 5
    (8, 4, 4, 70, 1100, 64),      # 280, 5
    (8, 8, 3, 61, 1100, 128),     # 183, 5
    (16, 8, 4, 50, 500, 128),     # 200, 9: the whole lane, rows of the cache and own ones
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bias", [None, "float", "half"])
@pytest.mark.parametrize("B,G,rep,T,rows,d", FORMS)
def test_trees_over_shares_of_many_tiles(B, G, rep, T, rows, d, bias, dtype):
    q, k, v, ck, cv = inputs(B, G, rep, T, rows, d, d, dtype, 3 * T + d)
    visible = tree_mask(T, 8)
    if bias:
        bias = torch.log(torch.floor(torch.rand(B, G, rows, generator=torch.Generator().manual_seed(4)) * 63 + 1)).to(
            torch.float32 if bias == "float" else dtype).cuda()
    scale = d ** -0.5
    out = log_kv_tree_attention(q, k, v, ck, cv, rows, visible.cuda(), scale, bias=bias)
    assert torch.equal(out, log_kv_tree_attention(q, k, v, ck, cv, rows, visible.cuda(), scale, bias=bias))
    for lane in ((0, 0), (B - 1, G - 1), (B // 2, G // 2)):
        for t in (0, T // 2, T - 1):
            check_token(out, q, k, v, ck, cv, lane, rows, t, visible[t].nonzero().flatten().cuda(), scale, bias)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,G,rep,T,rows,d", [(4, 8, 2, 300, 900, 128), (2, 8, 4, 300, 1100, 64), (8, 8, 4, 50, 700, 128)])
def test_causal_chunks_over_shares_of_many_tiles(B, G, rep, T, rows, d, dtype):
    """More than 128 queries of a KV group: 10, 8 and 4 tiles a share, own tiles behind the cache's among them."""
    q, k, v, ck, cv = inputs(B, G, rep, T, rows + T, d, d, dtype, 7 * T + d)
    w, scale = torch.zeros(B, G, rows + T, device="cuda"), d ** -0.5
    state = [x.clone() for x in (ck, cv, w)]
    out = log_kv_weight_attention(q, k, v, ck, cv, w, rows, scale)
    again = log_kv_weight_attention(q, k, v, *state, rows, scale)
    assert torch.equal(out, again) and all(torch.equal(x, y) for x, y in zip((ck, cv, w), state))
    for lane in ((0, 0), (B - 1, G - 1)):
        for t in (0, 63, 64, T // 2, T - 1) if T > 64 else (0, T // 2, T - 1):
            check_token(out, q, k, v, ck, cv, lane, rows, t, torch.arange(t + 1, device="cuda"), scale)
