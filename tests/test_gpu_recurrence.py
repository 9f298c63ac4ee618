"""GPU: the gated linear recurrence (mz_linear_recurrence, mz_linear_recurrence_backward) against a float64 loop: sizes from one
position to several blocks of positions, odd sizes, strides, every element type, gradients against the formula and against
differences, continuation step by step, captured graphs, other streams, and the lambda returns of a move log.

Tolerance: y[t] is a sum of products of at most t gates with one input; in any order of evaluation each term meets at most
2 T + 2 roundings of the arithmetic (u = 2^-24, or 2^-53), so |error| <= (2 T + 2) u z[t] with z the same recurrence over
absolute values, plus half a unit of the stored type.  A gate's gradient multiplies two such values, one of them as stored."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def wide(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def loop(a, x, state, reverse):
    """(y, last) in float64 on the host."""
    a, x = a.detach().double().cpu(), x.detach().double().cpu()
    h = torch.zeros(x.shape[0], x.shape[2], dtype=torch.float64) if state is None else state.detach().double().cpu().clone()
    y = torch.empty(x.shape, dtype=torch.float64)
    for t in (reversed(range(x.shape[1])) if reverse else range(x.shape[1])):
        h = a[:, t] * h + x[:, t]
        y[:, t] = h
    return y, h


def loop_backward(a, y, state, dy, dlast, reverse):
    """(dx, dgate, dstate) in float64 on the host, by the formula."""
    a, dy = a.detach().double().cpu(), dy.double().cpu()
    B, T, D = dy.shape
    order = list(reversed(range(T))) if reverse else list(range(T))
    g = torch.zeros(B, D, dtype=torch.float64) if dlast is None else dlast.double().cpu().clone()
    h0 = torch.zeros(B, D, dtype=torch.float64) if state is None else state.detach().double().cpu()
    dx, da = torch.empty_like(dy), torch.empty_like(dy)
    for i in range(T - 1, -1, -1):
        t = order[i]
        g = g + dy[:, t]
        dx[:, t] = g
        da[:, t] = g * (y[:, order[i - 1]] if i else h0)
        g = a[:, t] * g
    return dx, da, g


def inputs(B, T, D, dtype, seed=0, cuts=True):
    g = torch.Generator().manual_seed(seed)
    a = torch.sigmoid(torch.randn(B, T, D, generator=g) * 2 + 2)
    if cuts:
        a = torch.where(torch.rand(B, T, D, generator=g) < 0.03, torch.zeros(()), a)
    a = a * torch.where(torch.rand(B, T, D, generator=g) < 0.2, -1.0, 1.0)
    x = torch.randn(B, T, D, generator=g)
    s = torch.randn(B, D, generator=g)
    return a.to(dtype).cuda(), x.to(dtype).cuda(), s.to(wide(dtype)).cuda()


def close(got, want, z, T, dtype, extra=0.0):
    u = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    half = torch.finfo(got.dtype).eps / 2
    tol = (2 * T + 2) * u * z + half * want.abs() * (1 + 2 ** -6) + torch.finfo(got.dtype).tiny * 1.0 + extra
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25          # half a step of its subnormal numbers
    bad = (got.double().cpu() - want).abs() > tol
    assert got.shape == want.shape and not bad.any(), (int(bad.sum()), bad.nonzero()[:3])


SHAPES = [(1, 1, 1), (3, 1, 5), (64, 1, 130), (2, 7, 64), (1, 255, 3), (5, 257, 33), (2, 1000, 66), (1, 129, 257), (300, 40, 1),
          (7, 4097, 1), (1, 9001, 2), (3, 513, 128), (1, 2, 1000), (2, 128, 64), (1, 70000, 1), (5000, 1, 1), (999, 5, 1)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_forward_and_gradients(shape, dtype):
    from muzero_amd.targets import linear_recurrence
    B, T, D = shape
    for reverse in (False, True):
        for with_state in (False, True):
            a, x, s = inputs(B, T, D, dtype, seed=T + D)
            s = s if with_state else None
            y_ref, last_ref = loop(a, x, s, reverse)
            z, zl = loop(a.abs(), x.abs(), None if s is None else s.abs(), reverse)
            y, last = linear_recurrence(a, x, s, reverse=reverse)
            assert y.dtype == dtype and last.dtype == wide(dtype)
            close(y, y_ref, z, T, dtype)
            close(last, last_ref, zl, T, dtype)
            leaves = [t.clone().requires_grad_() for t in (a, x) + ((s,) if with_state else ())]
            y2, last2 = linear_recurrence(leaves[0], leaves[1], leaves[2] if with_state else None, reverse=reverse)
            assert torch.equal(y, y2) and torch.equal(last, last2)
            g = torch.Generator().manual_seed(9)
            dy = torch.randn(B, T, D, generator=g).to(dtype).cuda()
            dlast = torch.randn(B, D, generator=g).to(wide(dtype)).cuda()
            for use in (None, dlast):
                grads = torch.autograd.grad((y2, last2) if use is not None else (y2,), leaves,
                                            (dy, use) if use is not None else (dy,), retain_graph=True)
                dx_ref, da_ref, ds_ref = loop_backward(a, y_ref, s, dy, use, reverse)
                zx, zda, zs = loop_backward(a.abs(), z, None if s is None else s.abs(), dy.abs(), None if use is None else use.abs(), reverse)
                close(grads[1], dx_ref, zx, T, dtype)
                half = torch.finfo(dtype).eps / 2
                close(grads[0], da_ref, 2 * zda, T, dtype, extra=half * zda + (2.0 ** -25 * zx if dtype == torch.float16 else 0.0))
                if with_state:
                    close(grads[2], ds_ref, zs, T + 1, dtype)


def test_gradient_against_differences():
    from muzero_amd.targets import linear_recurrence
    a, x, s = (t.requires_grad_() for t in inputs(2, 9, 3, torch.float64, cuts=False))
    for reverse in (False, True):
        assert torch.autograd.gradcheck(lambda *v: linear_recurrence(*v, reverse=reverse), (a, x, s))


@pytest.mark.parametrize('dtype', TYPES)
def test_strides(dtype):
    """Every layout gives the bits of the contiguous call, or stays within the tolerance where another kernel serves it."""
    from muzero_amd.targets import linear_recurrence
    B, T, D = 3, 150, 34
    a, x, s = inputs(B, T, D, dtype, seed=3)
    y_ref, _ = loop(a, x, s, False)
    z, _ = loop(a.abs(), x.abs(), s.abs(), False)
    room = torch.zeros(B, T + 3, D + 5, dtype=dtype, device='cuda')
    sliced = room[:, 2:-1, 1:-4]                       # odd strides, pointers off by one element
    sliced.copy_(x)
    by_time = x.transpose(0, 1).contiguous().transpose(0, 1)
    by_channel = x.transpose(1, 2).contiguous().transpose(1, 2)
    odd = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    for xi in (sliced, by_time, by_channel, odd):
        for ai in (a, a.transpose(1, 2).contiguous().transpose(1, 2)):
            close(linear_recurrence(ai, xi, s)[0], y_ref, z, T, dtype)
            leaf = xi.detach().requires_grad_()
            y, _ = linear_recurrence(ai, leaf, s)
            g, = torch.autograd.grad(y.sum(), leaf)    # an expanded gradient
            dx, _, _ = loop_backward(a, y_ref, s, torch.ones(B, T, D), None, False)
            zx, _, _ = loop_backward(a.abs(), z, s, torch.ones(B, T, D), None, False)
            close(g, dx, zx, T, dtype)
    assert (room[:, :2] == 0).all() and (room[:, -1] == 0).all()
    # time-major rows of one channel: [T, B] as a move log holds them
    tm = x[:, :, 0].t().contiguous().t()[:, :, None]
    at = a[:, :, 0].t().contiguous().t()[:, :, None]
    close(linear_recurrence(at, tm, s[:, :1].contiguous())[0], y_ref[:, :, :1], z[:, :, :1], T, dtype)


def test_broadcast_gate_and_its_gradient():
    from muzero_amd.targets import linear_recurrence
    B, T, D = 4, 37, 20
    _, x, _ = inputs(B, T, D, torch.float32)
    for shape in ((1, 1, 1), (1, 1, D), (B, T, 1), (1, T, 1)):
        gate = torch.rand(shape, device='cuda').requires_grad_()
        y, _ = linear_recurrence(gate.expand(B, T, D), x)
        y_ref, _ = loop(gate.expand(B, T, D), x, None, False)
        z, _ = loop(gate.expand(B, T, D), x.abs(), None, False)
        close(y, y_ref, z, T, torch.float32)
        g, = torch.autograd.grad(y, gate, torch.ones_like(y))
        _, da, _ = loop_backward(gate.expand(B, T, D), y_ref, None, torch.ones(B, T, D), None, False)
        _, zda, _ = loop_backward(gate.expand(B, T, D), z, None, torch.ones(B, T, D), None, False)
        want = da.sum_to_size(shape)
        # the sum over a broadcast axis adds at most B T D terms in float32
        tol = (4 * T + 8 + B * T * D) * 2.0 ** -24 * zda.sum_to_size(shape) + 1e-7
        assert ((g.double().cpu() - want).abs() <= tol).all()


def test_step_by_step_continues_the_record():
    from muzero_amd.targets import linear_recurrence
    a, x, s = inputs(5, 12, 70, torch.bfloat16)
    y, last = linear_recurrence(a, x, s)
    state, parts = s, []
    for t in range(12):
        yt, state = linear_recurrence(a[:, t:t + 1], x[:, t:t + 1], state)
        parts.append(yt)
    y_ref, last_ref = loop(a, x, s, False)
    z, zl = loop(a.abs(), x.abs(), s.abs(), False)
    close(torch.cat(parts, 1), y_ref, z, 12, torch.bfloat16)
    close(state, last_ref, zl, 12, torch.bfloat16)


def test_empty_records():
    from muzero_amd.targets import linear_recurrence
    for B, T, D in ((2, 0, 3), (0, 4, 3), (2, 4, 0)):
        a = torch.ones(B, T, D, device='cuda', requires_grad=True)
        x = torch.ones(B, T, D, device='cuda', requires_grad=True)
        s = torch.randn(B, D, device='cuda').requires_grad_()
        y, last = linear_recurrence(a, x, s)
        assert y.shape == (B, T, D) and torch.equal(last, s)
        grads = torch.autograd.grad((y, last), (a, x, s), (torch.ones_like(y), torch.ones_like(last)))
        assert torch.equal(grads[2], torch.ones_like(s))


def test_a_gate_of_zero_cuts_and_neighbours_stay_apart():
    """A cut keeps what lies before it out; a row with NaN or infinity leaves the other rows and channels alone."""
    from muzero_amd.targets import linear_recurrence
    a, x, _ = inputs(3, 600, 65, torch.float32, cuts=False)
    clean, _ = linear_recurrence(a, x)
    x2 = x.clone()
    x2[1, 5, 7], x2[1, 300, 40] = float('nan'), float('inf')
    y, _ = linear_recurrence(a, x2)
    keep = torch.ones(3, 65, dtype=torch.bool)
    keep[1, 7] = keep[1, 40] = False
    assert torch.equal(y.transpose(1, 2)[keep.cuda()], clean.transpose(1, 2)[keep.cuda()])
    assert torch.equal(y[1, :5, 7], clean[1, :5, 7]) and y[1, 5:, 7].isnan().all()
    a[:, 200] = 0.0
    x3 = x.clone()
    x3[:, :200] += 1.0
    assert torch.equal(linear_recurrence(a, x)[0][:, 200:], linear_recurrence(a, x3)[0][:, 200:])


@pytest.mark.parametrize('shape,dtype', [((4, 700, 96), torch.bfloat16), ((6, 5000, 1), torch.float32), ((1, 4000, 40), torch.float64)])
def test_captured_replayed_and_on_another_stream(shape, dtype):
    from muzero_amd.targets import linear_recurrence
    a, x, s = inputs(*shape, dtype)
    gx, ga = x.clone(), a.clone()
    linear_recurrence(ga, gx, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        linear_recurrence(ga, gx, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, last = linear_recurrence(ga, gx, s)
    for i in range(4):
        gx.copy_(x * (i + 1))
        graph.replay()
        want, wlast = linear_recurrence(a, x * (i + 1), s)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(last, wlast)
    with torch.cuda.stream(side):
        other, _ = linear_recurrence(a, x, s)
    side.synchronize()
    assert torch.equal(other, linear_recurrence(a, x, s)[0])


def test_lambda_returns_of_a_move_log():
    from muzero_amd.targets import MoveLog
    rng = np.random.default_rng(0)
    n, B = 40, 33
    log = MoveLog(n + 5, B, (1, 1, 4), 2, 'cuda')
    r, v = rng.normal(size=(n, B)), rng.normal(size=(n, B))
    done, players = rng.random((n, B)) < 0.1, rng.integers(0, 2, (n, B))
    log.rewards[:n], log.root_values[:n] = torch.as_tensor(r), torch.as_tensor(v)
    log.done[:n], log.to_plays[:n] = torch.as_tensor(done.astype(np.uint8)), torch.as_tensor(players.astype(np.int32))
    log.rows = n
    boot = rng.normal(size=B)
    for gamma, lam, b in ((0.997, 0.9, None), (1.0, 1.0, boot), (0.9, 0.0, boot)):
        got = log.lambda_returns(gamma, lam, None if b is None else torch.as_tensor(b)).cpu().numpy()
        want = np.zeros((n, B))
        for k in range(n - 1, -1, -1):
            for e in range(B):
                if done[k, e]:
                    want[k, e] = r[k, e]
                elif k == n - 1:
                    want[k, e] = r[k, e] + gamma * (0.0 if b is None else b[e])
                else:
                    s = 1.0 if players[k, e] == players[k + 1, e] else -1.0
                    want[k, e] = r[k, e] + gamma * s * ((1 - lam) * v[k + 1, e] + lam * want[k + 1, e])
        np.testing.assert_allclose(got, want, rtol=0, atol=(6 * n + 8) * 2.0 ** -53 * 5 * n)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1, 769, 3), (2, 1500, 130), (1, 3000, 66), (3, 2049, 40), (1, 6000, 514)])
def test_chains_of_links(shape, dtype):
    """Long records of few channels: right, the same bits every time, and so when two calls run at once on two streams."""
    from muzero_amd.targets import linear_recurrence
    B, T, D = shape
    a, x, s = inputs(B, T, D, dtype, seed=T)
    dy = torch.randn(B, T, D, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    for reverse in (False, True):
        y_ref, last_ref = loop(a, x, s, reverse)
        z, zl = loop(a.abs(), x.abs(), s.abs(), reverse)
        y, last = linear_recurrence(a, x, s, reverse=reverse)
        close(y, y_ref, z, T, dtype)
        close(last, last_ref, zl, T, dtype)
        leaves = [t.clone().requires_grad_() for t in (a, x, s)]
        first = None
        for _ in range(3):
            y2, last2 = linear_recurrence(*leaves, reverse=reverse)
            grads = torch.autograd.grad(y2, leaves, dy)
            assert torch.equal(y, y2) and torch.equal(last, last2)
            first = first or grads
            assert all(torch.equal(g, f) for g, f in zip(grads, first))
        dx_ref, _, ds_ref = loop_backward(a, y_ref, s, dy, None, reverse)
        zx, _, zs = loop_backward(a.abs(), z, s.abs(), dy.abs(), None, reverse)
        close(first[1], dx_ref, zx, T, dtype)
        close(first[2], ds_ref, zs, T + 1, dtype)
        streams, outs = [torch.cuda.Stream() for _ in range(2)], []
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            for st in streams:
                with torch.cuda.stream(st):
                    outs.append(linear_recurrence(a, x, s, reverse=reverse))
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        assert all(torch.equal(o, y) and torch.equal(l, last) for o, l in outs)


@pytest.mark.parametrize('dtype', TYPES)
def test_long_rows(dtype):
    """Rows of one channel cut into links, and channels contiguous in time: right, and the same bits every time."""
    from muzero_amd.targets import linear_recurrence
    for B, T, D in ((2, 16385, 1), (1, 24577, 3)):
        a, x, s = inputs(B, T, D, dtype, seed=T)
        dy = torch.randn(B, T, D, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
        rows = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()  # noqa: E731
        for reverse in (False, True):
            y_ref, last_ref = loop(a, x, s, reverse)
            z, zl = loop(a.abs(), x.abs(), s.abs(), reverse)
            dx_ref, da_ref, ds_ref = loop_backward(a, y_ref, s, dy, s, reverse)
            zx, zda, zs = loop_backward(a.abs(), z, s.abs(), dy.abs(), s.abs(), reverse)
            first = None
            for _ in range(3):
                leaves = (rows(a), rows(x), s.clone().requires_grad_())
                y, last = linear_recurrence(*leaves, reverse=reverse)
                out = (y, last) + torch.autograd.grad((y, last), leaves, (rows(dy).detach(), s))
                first = first or out
                assert all(torch.equal(p, q) for p, q in zip(out, first))
            close(first[0], y_ref, z, T, dtype)
            close(first[1], last_ref, zl, T, dtype)
            close(first[3], dx_ref, zx, T, dtype)
            close(first[4], ds_ref, zs, T + 1, dtype)
            half = torch.finfo(dtype).eps / 2
            close(first[2], da_ref, 2 * zda, T, dtype, extra=half * zda + (2.0 ** -25 * zx if dtype == torch.float16 else 0.0))


def test_offsets_beyond_32_bits():
    """Sequences, positions and channels whose distance in memory passes 2^31 elements."""
    from muzero_amd.targets import linear_recurrence
    big = 2 ** 31 + 64
    room = torch.empty(2 * big + 70000, dtype=torch.bfloat16, device='cuda')
    for shape, strides in (((2, 300, 64), (big, 64, 1)), ((2, 3, 64), (big, 64, 1)), ((1, 3, 64), (0, big, 1)), ((2, 1000, 8), (big, 8, 1)),
                           ((2, 700, 1), (big, 1, 1)), ((1, 500, 3), (0, 1, big))):
        B, T, D = shape
        a, x, _ = inputs(B, T, D, torch.bfloat16, seed=T)
        far = room.as_strided(shape, strides, 8)
        far.copy_(x)
        y, last = linear_recurrence(a, far)
        y_ref, last_ref = loop(a, x, None, False)
        z, zl = loop(a.abs(), x.abs(), None, False)
        close(y, y_ref, z, T, torch.bfloat16)
        close(last, last_ref, zl, T, torch.bfloat16)


def test_refusals():
    from muzero_amd.targets import linear_recurrence
    t = torch.zeros(2, 3, 4, device='cuda')
    s = torch.zeros(2, 4, device='cuda')
    for args in ((t[0], t[0]), (t, t[:1]), (t, t.half()), (t.int(), t.int()), (t, t, s.double()), (t, t, s[:1]), (t, t, s.cpu()),
                 (t.half(), t.half(), s.half()), (t.double(), t.double(), s)):
        with pytest.raises(ValueError, match='linear_recurrence'):
            linear_recurrence(*args)
    x = t.clone().requires_grad_()
    y, _ = linear_recurrence(t, x)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)                 # differentiable once
    gate = t.clone().requires_grad_()
    y, _ = linear_recurrence(gate, x)
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(y.sum(), gate)
