"""Paged attention over rows wider than 128 features for many queries, whose tiles wait in LDS: own rows, prefixes, both,
masks, biases and what is not finite, against attention in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from harness import to_np  # noqa: F401
from paged_reference import dense, joined, joined_bias
from row_reference import check_close, reference, tree_mask
from test_gpu_paged_attention import Case, causal, make

pytestmark = pytest.mark.gpu

CASES = [
    # B, H, G, T, dk, dv, page, lengths, shared
    (8, 16, 8, 80, 256, 256, 16, [100, 0, 31, 32, 33, 7, 64, 1], None),
    (8, 16, 8, 80, 192, 128, 32, [0, 5, 100, 64, 96, 97, 31, 1], [150]),
    (6, 16, 8, 50, 136, 256, 16, [3 * b for b in range(6)], [40, 0, 129]),
    (4, 8, 8, 130, 200, 72, 64, [0] * 4, [1, 64]),
    (32, 16, 8, 4, 256, 256, 16, [11 * (b % 5) for b in range(32)], [1000]),
    (2, 1, 1, 700, 160, 144, 16, [500, 3], None),
]


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:7])))
def test_causal(case, dtype):
    Case(*case, dtype=dtype).check()


@pytest.mark.parametrize("case", [CASES[0], CASES[2]], ids=lambda c: "-".join(map(str, c[:7])))
def test_padded_batches_and_trees(case):
    B, T = case[0], case[3]
    c = Case(*case, seed=3)
    counts = torch.tensor([max(0, T - 9 * b) if b else T for b in range(B)], dtype=torch.int32, device="cuda")
    counts[-1] = 0
    c.check("counts", counts=counts)
    c.check("trees", visible=torch.stack([tree_mask(T, 5 + b, empty=(T - 1,)) for b in range(B)]).cuda())


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_prefix_of_rows_with_a_bias(dtype):
    from logkv_amd import SharedPrefix

    B, H, G, T, dk, dv, rows, N = 6, 16, 8, 50, 256, 192, 150, 2
    c = Case(B, H, G, T, dk, dv, 16, [7 * b for b in range(B)], dtype=dtype, seed=N)
    pk, pv = make(N, G, rows, dk + 8, dtype, 20)[..., :dk], make(N, G, rows, dv, dtype, 21)
    bias = (2 * torch.rand(N, G, rows, generator=torch.Generator().manual_seed(22))).cuda()
    bias[:, :, ::7] = -math.inf
    sizes = [rows, 77]
    for b, scale in ((bias, 1.0), (bias.to(dtype), 0.25), (None, 1.0)):
        got = c(prefix=SharedPrefix(torch.tensor(sizes, dtype=torch.int32, device="cuda"), k=pk, v=pv, bias=b, bias_scale=scale))
        (ck, total), (cv, _) = (joined((dense(p, c.table, c.lengths, max(c.lengths)), c.lengths), (x.cpu(), sizes), B)
                                for p, x in ((c.kp, pk), (c.vp, pv)))
        jb = None if b is None else joined_bias(b, sizes, c.lengths, ck.size(2), scale)
        out, _, bound, _ = reference(c.q, c.k, c.v, ck, cv, total, causal(B, T), c.scale, bias=jb)
        check_close(got, out, bound, scale)


def test_what_unused_slots_and_hidden_rows_hold():
    for dtype in (torch.bfloat16, torch.float16):
        for shared in ([75], None):
            T, lengths = 80, [17, 1, 50, 33]
            c = Case(4, 16, 8, T, 192, 192, 32, lengths, shared, dtype=dtype, seed=1, fill=float("nan"))
            c.check("unused slots")
            c.k[0, :, T - 1], c.v[0, :, T - 1] = float("nan"), float("inf")
            c.v[1, :, T - 1, 0] = -float("inf")
            c.check("hidden rows")
            if shared:
                c.vp[c.prefix_table[0, 0], :, 3, 1] = float("inf")
                c.vp[c.prefix_table[0, 1], :, 4, 2] = float("nan")
                c.check("infinities of the prefix")
            c.vp[c.table[3, 0], :, 0, 190] = -float("inf")
            c.check("infinities of one sequence")
            c.table[2, 1] = -1
            c.check("a page of zeros")
