"""GPU: the recurrence's kernel over contiguous channels at grids that the other tests do not reach: strands of 64 lanes (512 tiles
of 64 lanes and more) and grids of a multiple of 8 blocks, whose tiles are dealt out in another order - forward, gradients, both
directions, with and without a first state, every type; values and tolerances as in test_gpu_recurrence."""
import pytest
import torch

from test_gpu_recurrence import TYPES, close, inputs, loop, loop_backward, wide

pytestmark = pytest.mark.gpu

# tiles (32 lanes, or 64 from 512 tiles of 64 lanes on) of 4- and 8-byte, of 16-bit channels
GRIDS = [(600, 20, 3),       # 600 x 1 of 64 lanes, a multiple of 8
         (520, 17, 130),     # 520 x 3 | 520 x 2 of 64 lanes
         (515, 9, 64),       # 515 of 64 lanes, no multiple of 8; 16-bit: 515 of 128 channels
         (8, 20, 33),        # 8 x 2 | 8 x 2 (odd: single channels) of 32 lanes
         (16, 140, 32),      # 16 of 32 lanes, several rounds
         (8, 300, 512),      # 8 x 16 | 8 x 8 of 32 lanes: forward no chain only at 256 tiles and more
         (40, 300, 512)]     # 640 of 32 lanes (320 of 64) | 320 of 32: long records walked by their blocks


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', GRIDS)
def test_forward_and_gradients(shape, dtype):
    from muzero_amd.targets import linear_recurrence
    B, T, D = shape
    a, x, s = inputs(B, T, D, dtype, seed=T + D)
    g = torch.Generator().manual_seed(2)
    dy, dlast = torch.randn(B, T, D, generator=g).to(dtype).cuda(), torch.randn(B, D, generator=g).to(wide(dtype)).cuda()
    for reverse in (False, True):
        for state in (None, s):
            leaves = [t.clone().requires_grad_() for t in (a, x) + (() if state is None else (state,))]
            y, last = linear_recurrence(leaves[0], leaves[1], None if state is None else leaves[2], reverse=reverse)
            grads = torch.autograd.grad((y, last), leaves, (dy, dlast))
            y_ref, last_ref = loop(a, x, state, reverse)
            z, zl = loop(a.abs(), x.abs(), None if state is None else s.abs(), reverse)
            close(y.detach(), y_ref, z, T, dtype)
            close(last.detach(), last_ref, zl, T, dtype)
            dx_ref, da_ref, ds_ref = loop_backward(a, y_ref, state, dy, dlast, reverse)
            zx, zda, zs = loop_backward(a.abs(), z, None if state is None else s.abs(), dy.abs(), dlast.abs(), reverse)
            close(grads[1], dx_ref, zx, T, dtype)
            close(grads[0], da_ref, 2 * zda, T, dtype, extra=2.0 ** -25 * zx if dtype == torch.float16 else 0.0)
            if state is not None:
                close(grads[2], ds_ref, zs, T + 1, dtype)
