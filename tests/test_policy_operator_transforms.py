"""Transformations of torch that go round the tensor operators' native calls must raise: a tangent that is dropped and a trace
that fills nothing would be silent.  CPU: at the native calls, which refuse before anything is launched; GPU: at the public ones."""
import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.fx.experimental.proxy_tensor import make_fx


def recurrence_args(device):
    return torch.rand(2, 3, 4, device=device), torch.rand(2, 3, 4, device=device), torch.rand(2, 4, device=device)


def distill_args(device):
    return (torch.rand(3, 9, device=device), torch.zeros(3, 2, dtype=torch.int64, device=device), torch.rand(3, 2, device=device),
            torch.ones(3, device=device), torch.ones(3, device=device))


def verify_args(device):
    return (torch.zeros(2, 1, dtype=torch.int64, device=device), torch.rand(2, 1, 5, device=device), torch.rand(2, 2, 5, device=device),
            torch.rand(2, 1, dtype=torch.float64, device=device), torch.rand(2, dtype=torch.float64, device=device))


def native():
    from muzero_amd import engine
    n = engine.torch_calls()
    return [(lambda *a: n.linear_recurrence(*a, False, 0), recurrence_args), (lambda *a: n.distillation_loss(*a, 1.0, 0), distill_args),
            (lambda *a: n.distillation_loss_grad(*a, 1.0, 0), distill_args), (lambda *a: n.verify_drafts(*a, None, 0), verify_args)]


def public():
    from muzero_amd.drafts import verify_drafts
    from muzero_amd.targets import linear_recurrence
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    return [(lambda a, x, s: linear_recurrence(a, x, s), recurrence_args), (lambda z, i, t, e, w: distillation_loss(z, i, t, e, weight=w), distill_args),
            (lambda z, i, t, e, w: distillation_loss_grad(z, i, t, e, weight=w), distill_args),
            (lambda *a: verify_drafts(*a), verify_args)]


def check(calls, device):
    for call, make in calls:
        args = make(device)
        for i, t in enumerate(args):
            if not t.is_floating_point():
                continue
            with fwad.dual_level():
                dual = list(args)
                dual[i] = fwad.make_dual(t, torch.ones_like(t))
                with pytest.raises(NotImplementedError, match='forward-mode'):
                    call(*dual)
                with torch.no_grad(), pytest.raises(NotImplementedError, match='forward-mode'):
                    call(*dual)
        with pytest.raises(NotImplementedError, match='traced'):
            torch.jit.trace(call, args, check_trace=False)
        with pytest.raises(NotImplementedError, match='traced'):
            make_fx(call, tracing_mode='real')(*args)


def test_native_calls():
    check(native(), 'cpu')


@pytest.mark.gpu
def test_public_calls():
    check(public(), 'cuda')
    for call, make in public():
        call(*make('cuda'))             # and as before outside of such transformations
