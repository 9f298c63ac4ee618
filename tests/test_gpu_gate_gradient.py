"""GPU: a gate's gradient of 16-bit tensors is rounded once, like every other output of the recurrence: what precedes a position
enters it with more bits than the stored y has.

Tolerance: da = g * before; both carry at most 2 T + 2 roundings of float32 (z as in test_gpu_recurrence), the 8 bits kept of
what y's rounding lost leave at most one of their steps, 2^-15 (bfloat16) or 2^-18 (float16) of `before`, and da is rounded once:
half * (1 + 2^-6) of it covers both.  A float16 y among the subnormal numbers is off by up to 2^-25, times g."""
import pytest
import torch

from test_gpu_recurrence import close, inputs, loop, loop_backward

pytestmark = pytest.mark.gpu


def laid_out(t, layout):
    """The same values with channels, time or sequences contiguous."""
    order = {'channels': (0, 1, 2), 'time': (0, 2, 1), 'sequences': (1, 2, 0)}[layout]
    back = [order.index(i) for i in range(3)]
    return t.permute(*order).contiguous().permute(*back)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('shape,layout', [((64, 1, 136), 'channels'), ((6, 6, 136), 'channels'), ((3, 8, 64), 'channels'),
                                          ((5, 7, 33), 'channels'), ((1, 1501, 33), 'channels'), ((8, 200, 66), 'channels'),
                                          ((3, 300, 65), 'channels'), ((1, 1500, 130), 'channels'), ((2, 2049, 40), 'channels'),
                                          ((40, 300, 1), 'channels'), ((3, 77, 6), 'time'), ((4, 1000, 5), 'time'),
                                          ((1, 24577, 3), 'time'), ((33, 50, 1), 'sequences'), ((7, 1, 1), 'sequences')])
def test_rounded_once(shape, layout, dtype):
    from muzero_amd.targets import linear_recurrence
    B, T, D = shape
    a, x, s = inputs(B, T, D, dtype, seed=T)
    a, x = laid_out(a, layout), laid_out(x, layout)
    dy = laid_out(torch.randn(B, T, D, generator=torch.Generator().manual_seed(1)).to(dtype).cuda(), layout)
    for reverse in (False, True):
        y_ref, _ = loop(a, x, s, reverse)
        z, _ = loop(a.abs(), x.abs(), s.abs(), reverse)
        _, da_ref, _ = loop_backward(a, y_ref, s, dy, None, reverse)
        zx, zda, _ = loop_backward(a.abs(), z, s.abs(), dy.abs(), None, reverse)
        for up in (dy, laid_out(dy, 'channels')):     # the gradient may arrive in another layout than y has
            gate = a.detach().requires_grad_()
            y, _ = linear_recurrence(gate, x, s, reverse=reverse)
            da, = torch.autograd.grad(y, gate, up)
            close(da, da_ref, 2 * zda, T, dtype, extra=2.0 ** -25 * zx if dtype == torch.float16 else 0.0)


def test_values_at_the_ends_of_the_types():
    """Outputs of the largest and smallest numbers, infinity and NaN, where every record is cut and so y = x exactly."""
    from muzero_amd.targets import linear_recurrence
    for dtype, big in ((torch.float16, 65504.0), (torch.bfloat16, 3.3895e38)):
        tiny = torch.finfo(dtype).tiny / 64
        x = torch.tensor([1.0, big, -big, tiny, -tiny, 0.0, -0.0, 3.0, float('inf'), 1.0, 1.0, 1.0]).to(dtype).cuda()
        gate = torch.zeros(1, 12, 1, dtype=dtype, device='cuda', requires_grad=True)
        y, _ = linear_recurrence(gate, x[None, :, None])
        da, = torch.autograd.grad(y, gate, torch.ones_like(y))
        got = da[0, :, 0].float()
        assert torch.equal(got[1:9], x.float()[:8]) and got[0] == 0 and got[9] == float('inf') and got[10:].isnan().all()
    # a state beyond the type's range is stored as infinity, and so is what it gives the next gate
    gate = torch.ones(1, 3, 1, dtype=torch.float16, device='cuda', requires_grad=True)
    y, _ = linear_recurrence(gate, torch.full((1, 3, 1), 60000.0, dtype=torch.float16, device='cuda'))
    da, = torch.autograd.grad(y, gate, torch.full_like(y, 0.25))
    assert y[0, 1:].isinf().all() and da[0, 2].isinf().all() and da[0, 1, 0] == 30000.0


@pytest.mark.parametrize('shape', [(3, 300, 66), (1, 1500, 66), (9, 5, 8), (5, 600, 1)])
def test_a_captured_training_step(shape):
    """What the forward pass keeps for the gate's gradient is the captured pass's own, on every replay."""
    from muzero_amd.targets import linear_recurrence
    a, x, s = inputs(*shape, torch.bfloat16)
    dy = torch.randn(shape, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()

    def step(gate, x):
        y, last = linear_recurrence(gate, x, s)
        return (y, last) + torch.autograd.grad((y, last), (gate, x), (dy, s))

    leaves = lambda k: (a.clone().requires_grad_(), (x * k).requires_grad_())  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves(1))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g, z = leaves(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(g, z)
    for k in range(1, 5):
        with torch.no_grad():
            z.copy_(x * k)
        graph.replay()
        want = step(*leaves(k))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
