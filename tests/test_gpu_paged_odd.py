"""Infinities and NaNs in V of long caches: each reaches the queries that see its row, for about the time of the rows."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_paged_attention import Case, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("case", [
    # B, H, G, T, dk, dv, page, lengths, shared: streamed and tiled kernels, one and several blocks of queries
    (4, 2, 1, 1, 128, 128, 64, [700, 1, 63, 0], [900]),
    (2, 8, 2, 9, 64, 40, 16, [300, 0], [500, 333]),
    (2, 4, 1, 90, 128, 96, 16, [200, 130], [400]),
    (3, 2, 1, 150, 64, 64, 32, [500, 0, 333], None),
    (2, 4, 2, 40, 256, 200, 16, [150, 31], [260]),
    (2, 2, 1, 2, 192, 256, 16, [150, 31], [260])], ids=lambda c: "-".join(map(str, c[:7])))
def test_far_rows(case, dtype):
    """Of every kind, in the first and the last rows of a sequence's shares, in features at the ends of their words."""
    c = Case(*case, dtype=dtype, seed=4)
    dv, T = case[5], case[3]
    inf, nan = math.inf, math.nan
    last = max(range(len(c.lengths)), key=lambda b: c.lengths[b])

    def put(table, b, row, feature, value):
        c.vp[table[b, row // case[6]], :, row % case[6], feature] = value

    put(c.table, last, 0, 0, inf)
    put(c.table, last, c.lengths[last] - 1, dv - 1, -inf)
    put(c.table, last, c.lengths[last] // 2, 31, inf)
    put(c.table, last, c.lengths[last] // 2 + 1, 32, -inf)
    put(c.table, last, c.lengths[last] // 2 + 1, 31, -inf)      # both: NaN
    if c.shared:
        put(c.prefix_table, 0, c.shared[0] - 1, 33, nan)
        put(c.prefix_table, 0, 5, 0, inf)
        put(c.prefix_table, 0, 40, dv - 1, inf)
    c.check("cache rows")
    if T > 1:
        c.v[0, :, T - 1, 1], c.v[0, :, 1, 2], c.v[-1, :, 0, 3] = inf, -inf, nan
        c.check("the call's rows too")


def test_rows_hidden_by_a_bias():
    """What a row of a prefix holds that -inf hides reaches no query; beside it the same in rows that are seen."""
    from logkv_amd import SharedPrefix

    for T, H, half in ((1, 2, False), (90, 4, True)):
        c = Case(4, H, 1, T, 128, 128, 16, [40, 0, 3, 16], dtype=torch.bfloat16, seed=2)
        pk, pv = make(2, 1, 600, 128, torch.bfloat16, 5), make(2, 1, 600, 128, torch.bfloat16, 6)
        bias = torch.zeros(2, 1, 600, dtype=torch.bfloat16 if half else torch.float32, device="cuda")
        bias[:, :, 100:200] = -math.inf
        clean = c(prefix=SharedPrefix(600, k=pk, v=pv, bias=bias))
        pv[:, :, 100:200] = math.nan
        pv[0, :, 150] = math.inf
        assert torch.equal(c(prefix=SharedPrefix(600, k=pk, v=pv, bias=bias)), clean)
        pv[0, :, 201, 7] = -math.inf
        got = c(prefix=SharedPrefix(600, k=pk, v=pv, bias=bias))
        want = clean.clone()
        want[:2, :, :, 7] = -math.inf
        assert torch.equal(got, want)


def test_prefixes_of_a_call_differ():
    """Only the sequences behind a prefix see what it holds, also where shares go by length."""
    c = Case(6, 4, 1, 12, 128, 128, 16, [200, 3, 90, 0, 40, 150], [900, 3000, 0], seed=5)
    clean = c()
    c.vp[c.prefix_table[1, 2999 // 16], :, 2999 % 16, 64] = math.inf
    want = clean.clone()
    want[2:4, :, :, 64] = math.inf
    assert torch.equal(c(), want)
    c.vp[c.table[5, 0], :, 0, 127] = math.nan
    want[5, :, :, 127] = math.nan
    assert torch.equal(c().nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("T,H", [(1, 2), (40, 4)])
def test_time_of_long_rows(T, H):
    """One infinity among 2^19 rows costs a few times the call without it: no thread walks all rows."""
    from logkv_amd import SharedPrefix, log_kv_paged_attention

    rows, page, pages, d = 1 << 19, 64, 512, 64
    kp, vp = (make(pages, 1, page, d, torch.bfloat16, s) for s in (1, 2))
    line = (torch.arange(rows // page, dtype=torch.int32, device="cuda") % (pages - 1)).view(1, -1)
    line[0, -1] = pages - 1
    q, k, v = make(1, H, T, d, torch.bfloat16, 3, 2.0), make(1, 1, T, d, torch.bfloat16, 4), make(1, 1, T, d, torch.bfloat16, 5)
    own = line[:, :1].contiguous()

    def call(prefix):
        if prefix:
            return log_kv_paged_attention(q, k, v, kp, vp, own, 5, 0.125, prefix=SharedPrefix(rows, table=line))
        return log_kv_paged_attention(q, k, v, kp, vp, line, rows, 0.125)

    def ms(prefix):
        call(prefix)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call(prefix)
        end.record()
        end.synchronize()
        return start.elapsed_time(end)

    clean = [call(p) for p in (False, True)], [ms(p) for p in (False, True)]
    vp[pages - 1, :, page - 1, 9] = math.inf
    for p in (False, True):
        want = clean[0][p].clone()
        want[..., 9] = math.inf
        assert torch.equal(call(p), want)
        assert ms(p) < 20 * clean[1][p] + 2.0


@pytest.mark.parametrize("T,H", [(1, 2), (60, 4)])
def test_captured_while_values_come_and_go(T, H):
    """What a share left of its rows is read only beside that call's note: replays, two graphs and a side stream agree with
    eager calls while infinities appear in the pages and vanish."""
    c = Case(4, H, 1, T, 128, 128, 16, [33, 5, 600, 0], [700, 90])
    c()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c()
        graphs.append((graph, out))
    clean = c()
    places = [(c.prefix_table[0, 40], 3, 7, math.inf), (c.table[2, 30], 15, 64, -math.inf), (c.prefix_table[1, 2], 0, 0, math.nan), None]
    for place in places * 2:
        kept = c.vp.clone()
        if place is not None:
            page, slot, feature, value = place
            c.vp[page, :, slot, feature] = value
        want = c()
        assert torch.equal(want, clean) == (place is None)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = c()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in (beside, *(out for _, out in graphs)):
            assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(out.isnan(), want.isnan())
        c.vp.copy_(kept)
