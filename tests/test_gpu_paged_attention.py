"""Attention over a paged cache with shared prefixes on the GPU against the plain form in 64 bits."""

import math

import pytest
import torch

from paged_reference import dense, joined, joined_bias, pool
from row_reference import check_close, reference, tree_mask

pytestmark = pytest.mark.gpu


def make(B, H, T, d, dtype, seed, factor=1.0):
    return (factor * torch.randn(B, H, T, d, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def causal(B, T):
    return torch.ones(T, T, dtype=torch.bool).tril().expand(B, T, T)


class Case:
    """A call's tensors. ``shared``: rows of each prefix (in pages), None for no prefix."""

    def __init__(self, B, H, G, T, dk, dv, page, lengths, shared=None, dtype=torch.bfloat16, seed=0, fill=None):
        self.B, self.T, self.scale = B, T, dk ** -0.5
        self.q, self.k, self.v = (make(B, n, T, d, dtype, seed + i, 2.0 if i == 0 else 1.0)
                                  for i, (n, d) in enumerate(((H, dk), (G, dk), (G, dv))))
        self.lengths, self.shared = list(lengths), shared
        sizes = self.lengths + (list(shared) if shared else [])
        self.kp, self.vp, table = pool(len(sizes), G, dk, dv, page, sizes, dtype, seed + 7, "cuda", fill=fill)
        self.table = table[:B, :max(1, -(-max(self.lengths) // page))].contiguous()
        self.prefix_table = table[B:].contiguous() if shared else None
        self.n = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        self.pn = torch.tensor(list(shared), dtype=torch.int32, device="cuda") if shared else None

    def prefix(self):
        from logkv_amd import SharedPrefix

        return SharedPrefix(self.pn, table=self.prefix_table) if self.shared else None

    def __call__(self, **kw):
        from logkv_amd import log_kv_paged_attention

        kw.setdefault("prefix", self.prefix())
        return log_kv_paged_attention(self.q, self.k, self.v, self.kp, self.vp, self.table, self.n, self.scale, **kw)

    def want(self, visible=None, counts=None):
        rows = []
        for pages in (self.kp, self.vp):
            own = dense(pages, self.table, self.lengths, max(max(self.lengths), 1)), self.lengths
            pre = (dense(pages, self.prefix_table, self.shared, max(max(self.shared), 1)), self.shared) if self.shared else None
            rows.append(joined(own, pre, self.B))
        (ck, total), (cv, _) = rows
        see = causal(self.B, self.T) if visible is None else visible.cpu().expand(self.B, self.T, self.T)
        out, _, bound, _ = reference(self.q, self.k, self.v, ck, cv, total, see, self.scale, counts=counts)
        return out, bound

    def check(self, what="", **kw):
        out, bound = self.want(kw.get("visible"), kw.get("counts"))
        check_close(self(**kw), out, bound, what)


CASES = [
    # B, H, G, T, dk, dv, page, lengths, shared
    (1, 2, 1, 1, 64, 64, 16, [0], None),
    (2, 4, 2, 1, 128, 128, 16, [5, 100], None),
    (3, 6, 2, 5, 64, 32, 32, [31, 32, 33], None),
    (4, 2, 1, 1, 128, 128, 64, [0, 1, 63, 64], [100]),
    (4, 8, 2, 1, 128, 128, 16, [17, 0, 5, 40], [333, 16]),
    (6, 3, 1, 7, 80, 96, 16, [9, 70, 0, 15, 16, 17], [257, 1, 31]),
    (16, 4, 1, 1, 64, 64, 128, [3 * b for b in range(16)], [1000]),
    (8, 8, 2, 3, 128, 64, 16, [20] * 8, [511]),
    (2, 2, 1, 130, 64, 64, 32, [50, 0], [400]),
    (12, 8, 1, 2, 128, 128, 16, [7 * b for b in range(12)], [640, 200, 0]),
    (5, 5, 1, 1, 192, 128, 16, [30, 0, 16, 2, 77], [129]),
    (3, 2, 2, 20, 256, 256, 64, [10, 65, 0], [65, 0, 3]),
    (1, 1, 1, 3, 8, 8, 16, [2], [1]),
    (2, 2, 2, 1, 64, 128, 16, [0, 0], [0]),
    (3, 4, 4, 70, 128, 128, 16, [33, 100, 0], None),
]


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:7])))
def test_causal(case, dtype):
    Case(*case, dtype=dtype).check()


@pytest.mark.parametrize("case", [CASES[2], CASES[5], CASES[8], CASES[11]], ids=lambda c: "-".join(map(str, c[:7])))
def test_padded_batches_and_trees(case):
    B, T = case[0], case[3]
    for dtype in (torch.bfloat16, torch.float16):
        c = Case(*case, dtype=dtype, seed=3)
        counts = torch.tensor([max(0, T - 2 * b) if b else T for b in range(B)], dtype=torch.int32, device="cuda")
        counts[-1] = 0
        c.check("counts", counts=counts)
        trees = torch.stack([tree_mask(T, 5 + b, empty=(T - 1,)) for b in range(B)]).cuda()
        c.check("trees", visible=trees)
        c.check("one tree", visible=trees[0].contiguous())


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("B,H,G,T,dk,dv,rows,width", [
    (4, 4, 2, 1, 128, 128, 100, 136), (6, 4, 1, 3, 64, 64, 333, 72), (2, 2, 1, 90, 128, 128, 257, 128), (2, 3, 1, 5, 192, 64, 50, 200)])
def test_prefix_of_rows_with_a_bias(B, H, G, T, dk, dv, rows, width, dtype):
    """Packed rows whose log-mass stands in a column, hidden rows, and a factor."""
    from logkv_amd import SharedPrefix, log_kv_paged_attention

    for N in (1, 2):
        c = Case(B, H, G, T, dk, dv, 16, [3 * b for b in range(B)], dtype=dtype, seed=N)
        packed = make(N, G, rows, width + 8, dtype, 20)
        pk, pv = packed[..., :dk], make(N, G, rows, width, dtype, 21)[..., :dv]
        bias = (2 * torch.rand(N, G, rows, generator=torch.Generator().manual_seed(22))).cuda()
        bias[:, :, ::7] = -math.inf
        bias[:, :, 3] = -10000.0
        half = packed[..., width]
        sizes = [rows - 5 * i for i in range(N)]
        for b, scale in ((bias, 1.0), (bias, 0.25), (half, 1.0), (None, 1.0)):
            prefix = SharedPrefix(torch.tensor(sizes, dtype=torch.int32, device="cuda"), k=pk, v=pv, bias=b, bias_scale=scale)
            got = c(prefix=prefix)
            parts = []
            for pages, x in ((c.kp, pk), (c.vp, pv)):
                own = dense(pages, c.table, c.lengths, max(max(c.lengths), 1)), c.lengths
                parts.append(joined(own, (x.cpu(), sizes), B))
            (ck, total), (cv, _) = parts
            jb = None if b is None else joined_bias(b, sizes, c.lengths, ck.size(2), scale)
            out, _, bound, _ = reference(c.q, c.k, c.v, ck, cv, total, causal(B, T), c.scale, bias=jb)
            check_close(got, out, bound, (N, scale))
        # One length for all, given by the host.
        prefix = SharedPrefix(sizes[-1], k=pk, v=pv)
        same = SharedPrefix(torch.full((N,), sizes[-1], dtype=torch.int32, device="cuda"), k=pk, v=pv)
        assert torch.equal(c(prefix=prefix), c(prefix=same))


@pytest.mark.parametrize("shape", [(4, 2, 1, 1, 128, 128), (3, 4, 1, 20, 64, 64), (9, 8, 1, 1, 128, 64), (2, 2, 1, 3, 192, 192)],
                         ids=str)
def test_what_unused_slots_and_hidden_rows_hold(shape):
    """NaN in the pages' unused slots, in unused pages and in rows that a query does not see reaches no output; infinities
    that it sees do."""
    B, H, G, T, dk, dv = shape
    for dtype in (torch.bfloat16, torch.float16):
        for shared in ([75], None):
            lengths = [17 * b + 1 for b in range(B)]
            c = Case(B, H, G, T, dk, dv, 32, lengths, shared, dtype=dtype, seed=1, fill=float("nan"))
            c.check("unused slots")
            if T > 1:
                # The last call row is seen by the last query alone.
                c.k[0, :, T - 1], c.v[0, :, T - 1] = float("nan"), float("inf")
                c.v[1, :, T - 1, 0] = -float("inf")
                c.check("hidden rows")
            if shared:
                c.vp[c.prefix_table[0, 0], :, 3, 1] = float("inf")
                c.vp[c.prefix_table[0, 1], :, 4, 2] = float("nan")
                c.check("infinities of the prefix")
            c.vp[c.table[B - 1, 0], :, 0, 0] = -float("inf")
            c.check("infinities of one sequence")
            c.k[0, :, 0, 0] = float("nan")
            c.check("NaN logits of one sequence")


def test_entries_outside_the_pool_are_pages_of_zeros():
    for dtype, T, H in ((torch.bfloat16, 1, 2), (torch.float16, 3, 2), (torch.bfloat16, 40, 2)):
        c = Case(3, H, 1, T, 128, 128, 16, [50, 20, 33], [90], dtype=dtype)
        c.table[0, 1], c.table[2, 2], c.prefix_table[0, 2] = -1, c.kp.size(0), 2 ** 31 - 1
        c.check()
        c.kp, c.vp = c.kp[:0], c.vp[:0]
        c.check("an empty pool")


def test_lengths_beyond_the_table_are_held_to_it():
    c = Case(2, 2, 1, 2, 64, 64, 16, [32, 16], [48])
    want = c()
    c.n[0], c.pn[0] = 1000, 100000
    assert torch.equal(c(), want)
    c.n[1] = -5
    c.lengths = [32, 0]
    c.shared = [48]
    c.check()


def test_other_activation_dtypes_and_strides():
    for dtype in (torch.bfloat16, torch.float16):
        c = Case(2, 4, 2, 3, 64, 64, 16, [20, 5], [40], dtype=dtype)
        want = c()
        for x in ("q", "k", "v"):
            setattr(c, x, getattr(c, x).transpose(1, 2).contiguous().transpose(1, 2))
        assert torch.equal(c(), want)
        kp, vp = c.kp, c.vp
        both = torch.empty(kp.size(0), 16, 2, 2, 64, dtype=dtype, device="cuda")
        both[:, :, 0], both[:, :, 1] = kp.transpose(1, 2), vp.transpose(1, 2)
        c.kp, c.vp = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
        assert torch.equal(c(), want)
        c.q, c.k, c.v = c.q.float(), c.k.float(), c.v.float()
        got = c()
        assert got.dtype == torch.float32 and torch.equal(got.to(dtype), want)


def test_shares_by_length():
    """Prefixes and sequences of very different lengths, with many queries each."""
    c = Case(6, 4, 1, 12, 128, 128, 16, [2000, 3, 900, 0, 40, 1500], [3000, 100], seed=5)
    c.check()
    c = Case(3, 4, 1, 40, 64, 64, 64, [2500, 3, 900], dtype=torch.float16, seed=6)
    c.check()


def test_captured_twice_and_on_side_streams():
    c = Case(4, 4, 2, 2, 128, 128, 16, [33, 5, 60, 1], [200])
    room = Case(4, 4, 2, 2, 128, 128, 16, [64, 64, 64, 64], [208])
    c.kp, c.vp, c.table, c.prefix_table = room.kp, room.vp, room.table, room.prefix_table
    c()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c()
        graphs.append((graph, out))
    for step in range(4):
        c.q.normal_(generator=torch.Generator("cuda").manual_seed(step))
        c.n.copy_(torch.tensor([7 * step + 1, 16 * step, 64, 3]))
        c.pn.fill_(208 - 50 * step)
        c.lengths, c.shared = c.n.tolist(), c.pn.tolist()
        want = c()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = c()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(beside, want) and all(torch.equal(out, want) for _, out in graphs)
        c.check(step)


def test_two_calls_at_once():
    """Calls on two streams, each with its own scratch, give what they give alone."""
    cases = [Case(16, 8, 2, 1, 128, 128, 16, [200 + 7 * b for b in range(16)], [3000], seed=1),
             Case(6, 4, 1, 12, 128, 128, 16, [900, 3, 40, 0, 700, 64], [2000, 100], seed=2)]
    want = [c() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                got[i].append(c())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_rows_beyond_2_31_elements():
    """Pages and rows of a shared cache whose offsets pass 32 bits."""
    from logkv_amd import SharedPrefix, log_kv_paged_attention

    G, d, page, pages = 8, 128, 256, 8300                       # 2.18e9 elements
    kp = torch.zeros(pages, G, page, d, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros(pages, G, page, 8, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    for p in (pages - 1, pages - 2, 3):
        kp[p].normal_(generator=g), vp[p].normal_(generator=g)
    q, k, v = make(2, G, 1, d, torch.bfloat16, 1, 2.0), make(2, G, 1, d, torch.bfloat16, 2), make(2, G, 1, 8, torch.bfloat16, 3)
    table = torch.tensor([[pages - 1], [3]], dtype=torch.int32, device="cuda")
    pre = torch.tensor([[pages - 2]], dtype=torch.int32, device="cuda")
    out = log_kv_paged_attention(q, k, v, kp, vp, table, 200, d ** -0.5, prefix=SharedPrefix(250, table=pre))
    few = [x[[pages - 1, 3, pages - 2]].clone() for x in (kp, vp)]
    small = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    want = log_kv_paged_attention(q, k, v, *few, small, 200, d ** -0.5, prefix=SharedPrefix(250, table=small[:1] + 2))
    assert torch.equal(out, want)
    # Rows far behind the first of a contiguous prefix: one group's of a cache with 17 million rows between groups.
    far = kp.view(-1, d)[: 2 * 8_400_000].view(1, 2, 8_400_000, d)
    far_v = vp.view(-1, 8)[: 2 * 8_400_000].view(1, 2, 8_400_000, 8)
    near = [x[:, :, :300].clone() for x in (far, far_v)]
    q, k, v = (x[:, :2] for x in (q, k, v))
    out, want = (log_kv_paged_attention(q, k, v, few[0][:, :2], few[1][:, :2], small, 5, d ** -0.5, prefix=SharedPrefix(300, k=a, v=b))
                 for a, b in ((far, far_v), near))
    assert out.shape == want.shape and torch.isfinite(out).all()
    # A longer cache has more shares: equal within the rounding of their sums and of the output.
    assert ((out.double() - want.double()).abs() <= 2 * 2.0 ** -8 * want.double().abs() + 1e-4).all()


def test_masks_of_the_lowest_value():
    """A finite bias of the type's lowest value beside ordinary rows leaves them all the weight."""
    from logkv_amd import SharedPrefix

    for T, H in ((1, 2), (5, 4), (40, 2)):
        c = Case(4, H, 1, T, 64, 64, 16, [9, 0, 20, 16], dtype=torch.bfloat16)
        pk, pv = make(2, 1, 70, 64, torch.bfloat16, 5), make(2, 1, 70, 64, torch.bfloat16, 6)
        bias = torch.full((2, 1, 70), torch.finfo(torch.float32).min, device="cuda")
        hidden = c(prefix=SharedPrefix(70, k=pk, v=pv, bias=bias))
        c.shared = None
        out, bound = c.want()
        check_close(hidden, out, bound, T)
        bias[0, 0, 3] = 0.5
        hidden = c(prefix=SharedPrefix(70, k=pk, v=pv, bias=bias))
        rows = (pk[:, :, 3:4].cpu(), [1, 0]), (pv[:, :, 3:4].cpu(), [1, 0])
        own = [(dense(p, c.table, c.lengths, 20), c.lengths) for p in (c.kp, c.vp)]
        (ck, total), (cv, _) = (joined(a, b, 4) for a, b in zip(own, rows))
        add = joined_bias(torch.full((2, 1, 1), 0.5), [1, 0], c.lengths, ck.size(2))
        out, _, bound, _ = reference(c.q, c.k, c.v, ck, cv, total, causal(4, T), c.scale, bias=add)
        check_close(hidden, out, bound, T)


def test_append_then_attend():
    """Steps of a batch behind a shared prefix, as they are used: the new tokens stored and attended, the lengths
    advanced; against one causal attention over everything."""
    from logkv_amd import SharedPrefix, log_kv_paged_append, log_kv_paged_attention
    from paged_reference import inverse, rotate

    B, H, G, d, page, P, dtype = 3, 4, 2, 64, 16, 45, torch.bfloat16
    f = inverse(10000.0, d // 2)
    kp, vp, table = pool(B + 1, G, d, d, page, [64] * B + [P], dtype, 1, "cuda")
    own, pre = table[:B].contiguous(), table[B:, :3].contiguous()
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    prefix = SharedPrefix(P, table=pre)
    # The prefix is written by one sequence's append.
    xk, xv = make(1, G, P, d, dtype, 2), make(1, G, P, d, dtype, 3)
    log_kv_paged_append(xk, xv, kp, vp, pre, 0, frequencies=f.cuda())
    ks, vs, qs, outs = [], [], [], []
    for step, T in enumerate((5, 1, 1, 20, 1)):
        q, k, v = (make(B, n, T, d, dtype, 10 * step + i, 2.0 if n == H else 1.0) for i, n in enumerate((H, G, G)))
        q2, k2 = log_kv_paged_append(k, v, kp, vp, own, lengths, q=q, frequencies=f.cuda(), first=P)
        out = log_kv_paged_attention(q2, k2, v, kp, vp, own, lengths, d ** -0.5, prefix=prefix)
        lengths.add_(T)
        ks.append(k2), vs.append(v), qs.append(q2), outs.append(out)
        pos = (P + sum(x.size(2) for x in ks[:-1]) + torch.arange(T)).expand(B, T)
        from paged_reference import within
        within(q2, *rotate(q, f, pos))
    q, k, v, out = (torch.cat(x, dim=2) for x in (qs, ks, vs, outs))
    ck, cv = (dense(x, pre, [P], P).expand(B, -1, -1, -1) for x in (kp, vp))
    want, _, bound, _ = reference(q, k, v, ck, cv, [P] * B, causal(B, k.size(2)), d ** -0.5)
    check_close(out, want, bound)


def test_refusals():
    from logkv_amd import SharedPrefix, log_kv_paged_attention

    c = Case(4, 4, 2, 2, 64, 64, 16, [16] * 4, [32])
    rows = make(2, 2, 40, 64, torch.bfloat16, 9)
    good = dict(q=c.q, k=c.k, v=c.v, k_pages=c.kp, v_pages=c.vp, table=c.table, lengths=c.n, scale=0.125, prefix=c.prefix())
    P = SharedPrefix
    tree = torch.ones(2, 2, dtype=torch.bool, device="cuda")
    for change, kind in (
            (dict(q=c.q[0]), ValueError), (dict(q=c.q[:, :3]), ValueError), (dict(k=c.k[:, :1]), ValueError),
            (dict(v=c.v[:, :, :1]), ValueError), (dict(q=c.q[..., :32]), ValueError), (dict(q=c.q.cpu()), ValueError),
            (dict(k_pages=c.kp[:, :, :8], v_pages=c.vp[:, :, :8]), ValueError), (dict(k_pages=c.kp.float(), v_pages=c.vp.float()), ValueError),
            (dict(v_pages=c.vp[1:]), ValueError), (dict(table=c.table.long()), ValueError), (dict(table=c.table[:2]), ValueError),
            (dict(lengths=17), ValueError), (dict(lengths=c.n[:2]), ValueError), (dict(scale=0.0), ValueError),
            (dict(scale=float("nan")), ValueError), (dict(visible=tree[:1]), ValueError), (dict(visible=tree.float()), ValueError),
            (dict(visible=tree, counts=c.n), ValueError), (dict(counts=c.n[:1]), ValueError),
            (dict(prefix=P(5)), ValueError), (dict(prefix=P(5, table=c.prefix_table, k=rows, v=rows)), ValueError),
            (dict(prefix=P(5, k=rows)), ValueError), (dict(prefix=P(41, k=rows, v=rows)), ValueError),
            (dict(prefix=P(5, table=c.prefix_table.expand(3, -1).contiguous())), ValueError),
            (dict(prefix=P(33, table=c.prefix_table)), ValueError), (dict(prefix=P(c.n, table=c.prefix_table)), ValueError),
            (dict(prefix=P(5, k=rows.float(), v=rows.float())), ValueError), (dict(prefix=P(5, k=rows[:, :1], v=rows[:, :1])), ValueError),
            (dict(prefix=P(5, k=rows, v=rows, bias=rows[..., 0, 0])), ValueError),
            (dict(prefix=P(5, k=rows, v=rows, bias=rows[..., 0], bias_scale=0.0)), ValueError),
            (dict(prefix=P(5, table=c.prefix_table, bias=rows[..., 0])), ValueError),
            (dict(prefix=P(5, k=rows[..., 1:, :].as_strided((2, 2, 39, 64), (4, 2, 1, 1)), v=rows[..., 1:, :])), ValueError),
            (dict(q=c.q.clone().requires_grad_()), NotImplementedError), (dict(q=c.q.double()), NotImplementedError)):
        with pytest.raises(kind):
            log_kv_paged_attention(**{**good, **change})
