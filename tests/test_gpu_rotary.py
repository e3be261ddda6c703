"""Rotary positions on the GPU against the formula in 64 bits, and their gradients."""

import pytest
import torch

from paged_reference import HALF, inverse, rotate, within

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def make(B, H, T, d, dtype, seed, strides="plain"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, T, d, generator=g).to(dtype).cuda()
    if strides == "tokens":       # [B, T, H, d] as a projection leaves it
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if strides == "fused":        # a part of wider rows, at an odd offset
        wide = torch.zeros(B, T, H * d + 3, dtype=dtype, device="cuda")
        view = wide[..., 3:].view(B, T, H, d).transpose(1, 2) if H * d else x
        view.copy_(x)
        return view
    if strides == "last":         # features not contiguous
        return x.transpose(2, 3).contiguous().transpose(2, 3)
    if strides == "expanded":
        return x[:1, :1].expand(B, H, T, d)
    return x


def positions_of(kind, B, T, seed):
    """(argument, [B, T])."""
    g = torch.Generator().manual_seed(seed)
    if kind == "first":
        return 7, (torch.arange(T) + 7).expand(B, T)
    if kind == "far":
        return (1 << 21) + 12345, (torch.arange(T) + (1 << 21) + 12345).expand(B, T)
    if kind == "negative":
        return -5, (torch.arange(T) - 5).expand(B, T)
    if kind == "line":
        p = torch.randint(0, 40000, (T,), generator=g)
        return p.cuda(), p.expand(B, T)
    p = torch.randint(0, 1 << 20, (B, 2 * T), generator=g, dtype=torch.int32)
    return p.cuda()[:, ::2], p[:, ::2]


@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,G,T,d,r", [
    (1, 2, 1, 1, 8, 8), (2, 3, 1, 5, 64, 64), (1, 16, 8, 1, 128, 128), (3, 4, 2, 33, 128, 64), (2, 2, 2, 7, 80, 20),
    (1, 5, 1, 9, 18, 18), (2, 1, 1, 3, 7, 2), (1, 2, 2, 4, 96, 48), (1, 1, 1, 2, 512, 512), (1, 2, 1, 3, 24, 0),
    (5, 3, 1, 1000, 40, 40), (1, 1, 1, 1, 1, 0), (2, 2, 2, 3, 256, 144)])
def test_rotation(B, H, G, T, d, r, dtype, interleaved):
    from logkv_amd import log_kv_rotary

    for n, (kind, strides) in enumerate((("first", "plain"), ("far", "tokens"), ("rows", "fused"), ("line", "last"),
                                         ("negative", "expanded"))):
        q, k = make(B, H, T, d, dtype, n, strides), make(B, G, T, d, dtype, 10 + n, strides)
        f = inverse(10000.0, r // 2)
        arg, pos = positions_of(kind, B, T, n)
        amplitude = 1.0 if n % 2 else 1.25
        got = log_kv_rotary(q, k, f.cuda(), arg, interleaved=interleaved, amplitude=amplitude)
        for x, y in zip((q, k), got):
            want, bound = rotate(x, f, pos, interleaved, amplitude)
            assert y.dtype == dtype and y.data_ptr() != x.data_ptr()
            within(y, want, bound, (kind, strides))


def test_many_tokens_and_one_input():
    from logkv_amd import log_kv_rotary

    q = make(3, 2, 3001, 64, torch.bfloat16, 1)
    f = inverse(500000.0, 32)
    out, none = log_kv_rotary(q, None, f.cuda(), 3)
    assert none is None
    within(out, *rotate(q, f, (torch.arange(3001) + 3).expand(3, -1)))


def test_float32_frequencies_and_half_exact():
    from logkv_amd import log_kv_rotary

    q = make(1, 2, 6, 32, torch.float32, 2)
    f = inverse(10000.0, 16).float()
    out, _ = log_kv_rotary(q, None, f.cuda(), 100)
    within(out, *rotate(q, f, (torch.arange(6) + 100).expand(1, -1)))
    # Position 0 leaves the features bit for bit.
    out, _ = log_kv_rotary(q, None, f.cuda(), torch.zeros(6, dtype=torch.int64, device="cuda"))
    assert torch.equal(out, q)


def test_tables_are_the_rotation():
    """The tables that a cache takes rotate as the operator does."""
    from logkv_amd import log_kv_rotary, rotary_frequencies, rotary_tables

    f, amplitude = rotary_frequencies(64, 10000.0, scaling=dict(kind="yarn", factor=4.0, original_max_seq_len=64))
    cos, sin = rotary_tables(f, 40, amplitude=amplitude)
    assert cos.shape == sin.shape == (40, 64) and cos.dtype == torch.float32
    q = make(1, 3, 40, 64, torch.float32, 3)
    out, _ = log_kv_rotary(q, None, f, amplitude=amplitude)
    rolled = torch.cat((-q[..., 32:], q[..., :32]), dim=-1)
    want = (q.double() * cos.double() + rolled.double() * sin.double()).cpu()
    within(out, want, rotate(q, f, torch.arange(40).expand(1, -1), amplitude=amplitude)[1] * 2 + 1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", (False, True))
def test_gradients(dtype, interleaved):
    """Against the formula (the rotation back), and against differences of the 64-bit rotation."""
    from logkv_amd import log_kv_rotary

    B, H, G, T, d, r = 2, 3, 1, 9, 40, 24
    f = inverse(10000.0, r // 2)
    pos = torch.randint(0, 100000, (B, T), generator=torch.Generator().manual_seed(4))
    q, k = (make(B, n, T, d, dtype, 5 + n, "tokens").requires_grad_() for n in (H, G))
    wq, wk = (make(B, n, T, d, dtype, 15 + n, "last") for n in (H, G))
    out = log_kv_rotary(q, k, f.cuda(), pos.cuda(), interleaved=interleaved, amplitude=1.5)
    dq, dk = torch.autograd.grad(out, (q, k), (wq, wk))
    for x, w, dx in ((q, wq, dq), (k, wk, dk)):
        want, bound = rotate(w, f, pos, interleaved, 1.5, sign=-1.0)
        within(dx, want, bound, "formula")
        # The map is linear: its difference along a direction is that direction's image.
        step = torch.randn(x.shape, generator=torch.Generator().manual_seed(6)).to(dtype)
        x0 = x.detach().cpu()
        y1 = rotate(x0.double().add(step.double()).float(), f, pos, interleaved, 1.5)[0]
        y0 = rotate(x0.float(), f, pos, interleaved, 1.5)[0]
        by_difference = float(((y1 - y0) * w.cpu().double()).sum())
        by_gradient = float((dx.cpu().double() * step.double()).sum())
        # The gradient's bound along the step, and the float32 rounding of the shifted point.
        slack = float((bound * step.double().abs()).sum()) + 1.5 * 2.0 ** -23 * float(
            (x0.double().abs() + step.double().abs()).sum() * w.cpu().double().abs().max())
        assert abs(by_difference - by_gradient) <= slack


def test_second_derivative_and_partial_gradients():
    from logkv_amd import log_kv_rotary

    f = inverse(10000.0, 4).cuda()
    q, k = (make(1, 2, 3, 8, torch.float32, n).requires_grad_(n == 1) for n in (1, 2))
    y, z = log_kv_rotary(q, k, f, 5)
    assert y.requires_grad and not z.requires_grad
    w = make(1, 2, 3, 8, torch.float32, 3).requires_grad_()
    (dq,) = torch.autograd.grad(y, q, w, create_graph=True)
    u = make(1, 2, 3, 8, torch.float32, 4)
    (dw,) = torch.autograd.grad(dq, w, u)     # the gradient's transpose: the rotation of u
    within(dw, *rotate(u, f, (torch.arange(3) + 5).expand(1, -1)))
    # A loss of keys alone, whose incoming gradient is an expanded one.
    k = make(1, 2, 3, 8, torch.float32, 2).requires_grad_()
    log_kv_rotary(q, k, f, 5)[1].sum().backward()
    within(k.grad, *rotate(torch.ones(1, 2, 3, 8), f, (torch.arange(3) + 5).expand(1, -1), sign=-1.0))
    assert q.grad is None
    with torch.no_grad():
        assert not log_kv_rotary(q, k, f, 5)[0].requires_grad


def test_empty_calls():
    from logkv_amd import log_kv_rotary

    f = inverse(10000.0, 4).cuda()
    for shape in ((0, 2, 3, 8), (1, 2, 0, 8)):
        q = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        y, z = log_kv_rotary(q, q, f)
        assert y.shape == z.shape == shape
    q, k = torch.zeros(1, 0, 3, 8, device="cuda"), make(1, 2, 3, 8, torch.float32, 1)
    within(log_kv_rotary(q, k, f)[1], *rotate(k, f, torch.arange(3).expand(1, -1)))


def test_infinities_stay_in_their_pair():
    from logkv_amd import log_kv_rotary

    f = inverse(10000.0, 8)
    q = make(1, 1, 4, 24, torch.bfloat16, 1)
    q[0, 0, 1, 2], q[0, 0, 2, 20] = float("nan"), float("inf")
    out = log_kv_rotary(q, None, f.cuda(), 3)[0].cpu()
    odd = ~torch.isfinite(out)
    assert odd.sum() == 3 and odd[0, 0, 1, 2] and odd[0, 0, 1, 10] and odd[0, 0, 2, 20]


def test_streams_devices_and_graphs():
    from logkv_amd import log_kv_rotary

    f = inverse(10000.0, 32).cuda()
    q, k, pos = make(2, 4, 8, 64, torch.bfloat16, 1), make(2, 2, 8, 64, torch.bfloat16, 2), torch.arange(8, device="cuda")
    want = log_kv_rotary(q, k, f, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = log_kv_rotary(q, k, f, pos)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, log_kv_rotary(q, k, f, pos)))
        graphs[-1] = (graph, graphs[-1][1])
    for step in range(4):
        pos.add_(1000 * step)
        q.normal_(generator=torch.Generator("cuda").manual_seed(step))
        want = log_kv_rotary(q, k, f, pos)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_captured_training_step():
    """Forward and gradient in one graph, replayed with the program's own work between."""
    from logkv_amd import log_kv_rotary

    f = inverse(10000.0, 32).cuda()
    q0, k0 = (make(2, n, 16, 64, torch.bfloat16, n) for n in (4, 2))
    wq, wk = (make(2, n, 16, 64, torch.bfloat16, 9 + n) for n in (4, 2))

    def step():
        q, k = (x.detach().requires_grad_() for x in (q0, k0))      # leaves that no earlier graph knows
        out = log_kv_rotary(q, k, f, 11)
        return (*out, *torch.autograd.grad(out, (q, k), (wq, wk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        q0.normal_(generator=torch.Generator("cuda").manual_seed(i))
        wk.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_gradient_of_changed_positions_is_refused():
    from logkv_amd import log_kv_rotary

    f, pos = inverse(10000.0, 16).cuda(), torch.arange(5, device="cuda")
    q = make(1, 2, 5, 32, torch.float32, 1).requires_grad_()
    for change in (lambda: pos.add_(1), lambda: f.mul_(2.0)):
        out, _ = log_kv_rotary(q, None, f, pos)
        out.sum().backward(retain_graph=True)
        change()
        with pytest.raises(RuntimeError, match="modified"):
            out.sum().backward()


def test_more_blocks_than_a_line_of_the_grid():
    from logkv_amd import log_kv_rotary

    T = (1 << 20) * 8 + 77      # 8 tokens a block
    f = torch.ones(1, dtype=torch.float64, device="cuda")
    q = torch.ones(2, 1, T, 2, dtype=torch.bfloat16, device="cuda")
    out, _ = log_kv_rotary(q, None, f)
    pos = torch.arange(T, device="cuda", dtype=torch.float64)
    want = torch.stack((pos.cos() - pos.sin(), pos.cos() + pos.sin()), dim=-1)
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -20
    for b in range(2):
        assert ((out[b, 0].double() - want).abs() <= bound).all()


def test_refusals():
    from logkv_amd import log_kv_rotary

    f = inverse(10000.0, 4).cuda()
    q, k = make(2, 2, 3, 8, torch.bfloat16, 1), make(2, 1, 3, 8, torch.bfloat16, 2)
    for args, kind in (
            ((q[0], k, f), ValueError), ((q, k[:1], f), ValueError), ((q, k[:, :, :2], f), ValueError),
            ((q, k.float(), f), ValueError), ((q, k.cpu(), f), ValueError), ((q.cpu(), k.cpu(), f), ValueError),
            ((q.to(torch.float64), None, f), NotImplementedError), ((q, k, f.cpu()), ValueError),
            ((q, k, f.to(torch.bfloat16)), ValueError), ((q, k, torch.cat((f, f))), ValueError), ((q, k, f[None]), ValueError),
            ((q, k, f, torch.arange(4, device="cuda")), ValueError), ((q, k, f, torch.arange(3)), ValueError),
            ((q, k, f, torch.arange(3, device="cuda").float()), ValueError), ((q, k, f, 1.5), TypeError),
            ((q, k, f.clone().requires_grad_()), NotImplementedError)):
        with pytest.raises(kind):
            log_kv_rotary(*args)
    with pytest.raises(ValueError):
        log_kv_rotary(q, k, f, amplitude=float("inf"))
    with pytest.raises(ValueError):
        log_kv_rotary(torch.zeros(1, 1, 1, 514, device="cuda"), None, f)


def test_bound_of_the_types():
    assert HALF == {t: torch.finfo(t).eps / 2 for t in HALF}
