"""GPU: the class of all actions outside the entries (teacher_lse), from a student that gives them much to one that gives them next
to nothing: loss and gradient against the definition in float64, taken from logarithms throughout.

Tolerance: a softmax sum is off by at most `rel` of itself - 2^-23 for every doubling between a term and what the sum is relative
to, averaged over the terms, for the exponential and its additions (16 + V / 64), and 24 more doublings for the outside sum, which
is relative to the row's maximum as long as it is no less than 2^-24.  The loss takes logarithms of two such sums, a gradient entry
two quotients, each output one rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def definition(logits, index, teacher, lse, tau, weight):
    z, t = logits.double().cpu() / tau, teacher.double().cpu() / tau
    R, V = z.shape
    at = index.cpu()
    w = weight.double().cpu()[:, None]
    inside = torch.zeros(R, V, dtype=torch.bool).scatter_(1, at, True)
    masked = ~inside & ((z == -math.inf) | (logits.cpu() == torch.finfo(logits.dtype).min))
    p = torch.zeros(R, V, dtype=torch.float64).scatter_(1, at, torch.exp(t - lse.double().cpu()[:, None]))
    logp = torch.full((R, V), -math.inf, dtype=torch.float64).scatter_(1, at, t - lse.double().cpu()[:, None])
    logq = z - torch.logsumexp(z, 1, keepdim=True)
    q, mass = logq.exp(), p.sum(1, keepdim=True)
    out = torch.where(inside | masked, -math.inf, logq)
    some = out.amax(1, keepdim=True) > -math.inf
    logrest = torch.logsumexp(out, 1, keepdim=True)
    rest = torch.where(some, (1 - mass).clamp(min=0), 0.0)
    qout = torch.where(some & (out > -math.inf), (out - torch.where(some, logrest, 0.0)).exp(), 0.0)
    kl = torch.where(p > 0, p * (logp - logq), 0.0).sum(1, keepdim=True)
    kl = kl + torch.where(rest > 0, torch.special.xlogy(rest, rest) - rest * torch.where(some, logrest, 0.0), 0.0)
    loss, grad = w * tau * tau * kl, w * tau * (q * (mass + rest) - p - rest * qout)
    doublings = lambda d: (d * math.log2(math.e)).nan_to_num(0, 0, 0).clamp(min=0, max=300)  # noqa: E731
    steps, osteps = doublings(logq.amax(1, keepdim=True) - logq), doublings(out.amax(1, keepdim=True) - out)
    rel = ((q * steps).sum(1, keepdim=True) + (qout * osteps).sum(1, keepdim=True) + 24 + 16 + V / 64) * 2.0 ** -23
    tol = (w * tau * tau).abs() * (mass + 2 * rest) * rel
    dtol = (w * tau).abs() * (q * (mass + rest) * (rel + (steps + 4) * 2.0 ** -23) + rest * qout * (rel + (osteps + 28) * 2.0 ** -23))
    return loss[:, 0], grad, tol[:, 0], dtol


def check(logits, index, teacher, lse, tau, weight):
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    want, dwant, tol, dtol = definition(logits, index, teacher, lse, tau, weight)
    loss, grad = distillation_loss_grad(logits, index, teacher, lse, tau, weight)
    leaf = logits.detach().requires_grad_()
    loss2 = distillation_loss(leaf, index, teacher, lse, tau, weight)
    up = torch.linspace(0.5, -2.0, len(loss), device='cuda')
    grad2, = torch.autograd.grad(loss2, leaf, up)
    half = torch.finfo(logits.dtype).eps / 2
    least = (2.0 ** -25 if logits.dtype == torch.float16 else 1e-37) + 1e-37 * float(weight.abs().max())
    for got in (loss, loss2):
        off = (got.double().cpu() - want).abs()
        assert (off <= tol + 2.0 ** -23 * want.abs()).all(), (got.cpu(), want)
    u = up.double().cpu()[:, None]
    for got, ref, dt in ((grad, dwant, dtol), (grad2, dwant * u, dtol * u.abs())):
        off = (got.double().cpu() - ref).abs()
        allowed = dt * (1 + half) + (half + 2.0 ** -23) * ref.abs() + least
        assert (off <= allowed).all(), ((off / allowed).max(), (off > allowed).nonzero()[:3])


def rows(V, K, gap, dtype, seed, masks):
    """Rows whose K entries stand `gap` above every other action; some of the others masked at -inf and at the lowest value."""
    g = torch.Generator().manual_seed(seed)
    R = 6
    z = torch.randn(R, V, generator=g)
    index = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(R)])
    z = (z - gap).scatter_(1, index, torch.randn(R, K, generator=g)).to(dtype)
    if masks:
        inside = torch.zeros(R, V, dtype=torch.bool).scatter_(1, index, True)
        low = torch.rand(R, V, generator=g)
        z = torch.where(~inside & (low < 0.3), torch.tensor(-math.inf, dtype=dtype), z)
        z = torch.where(~inside & (low > 0.8), torch.tensor(torch.finfo(dtype).min, dtype=dtype), z)
    return z.cuda(), index.cuda(), (torch.rand(R, generator=g) + 0.5).cuda(), g


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V,K', [(3, 1), (9, 4), (16, 16), (40, 7), (300, 12), (3000, 70), (9001, 5), (70001, 20)])
def test_from_much_to_next_to_nothing(V, K, dtype):
    for gap in (0.0, 10.0, 16.0, 17.0, 40.0, 80.0, 88.0, 110.0, 300.0, 3000.0):
        for tau in (1.0, 0.125, 4.0):
            for masks in (False, True):
                z, index, weight, g = rows(V, K, gap, dtype, V + int(gap), masks)
                teacher = torch.randn(len(z), K, generator=g).to(dtype).cuda()
                lse = torch.logsumexp(teacher.float() / tau, 1) + 0.3          # the entries hold exp(-0.3) of the teacher's mass
                check(z, index, teacher, lse, tau, weight)


def test_one_entry_above_a_low_tail():
    """[0, -g, -g - 5] with 0.7 on the first action: the loss grows with g without a jump and the gradient stays +-0.3."""
    from muzero_amd.trainer import distillation_loss_grad
    gaps = torch.tensor([20.0, 80.0, 86.0, 87.0, 88.0, 89.0, 110.0, 300.0, 60000.0])
    z = torch.stack([torch.zeros(9), -gaps, -gaps - 5], 1).cuda()
    index, teacher = torch.zeros(9, 1, dtype=torch.int64).cuda(), torch.zeros(9, 1).cuda()
    lse = torch.full((9,), -math.log(0.7)).cuda()
    loss, grad = distillation_loss_grad(z, index, teacher, lse)
    rest = 1 - math.exp(-lse[0].double().item())
    want = (1 - rest) * math.log(1 - rest) + rest * (math.log(rest) + gaps.double() - math.log1p(math.exp(-5)))
    assert ((loss.double().cpu() - want).abs() <= 2.0 ** -19 + 2.0 ** -23 * want).all()
    assert torch.allclose(grad[:, 0], torch.full((9,), rest).cuda(), rtol=1e-5)
    assert torch.allclose(grad.sum(1), torch.zeros(9).cuda(), atol=1e-6)


@pytest.mark.parametrize('V', [9, 50, 700, 20001])
def test_scaled_losses_stay_finite(V):
    """Large weights over a tail that is almost nothing, beside masked actions: no infinity on the way, no NaN."""
    for gap in (12.0, 25.0, 60.0, 87.0, 200.0):
        z, index, _, g = rows(V, 3, gap, torch.float32, V, True)
        teacher = torch.randn(6, 3, generator=g).cuda()
        lse = torch.logsumexp(teacher, 1) + 1.0
        check(z, index, teacher, lse, 1.0, torch.full((6,), 2.0 ** 24).cuda())


@pytest.mark.parametrize('V', [6, 33, 500, 30000])
def test_everything_outside_masked(V):
    """Nothing outside that the student plays: the class is left out, whether the mask is -inf or the type's lowest value."""
    from muzero_amd.trainer import distillation_loss_grad
    for dtype in TYPES:
        for low in (-math.inf, torch.finfo(dtype).min):
            z = torch.full((4, V), low, dtype=dtype).cuda()
            z[:, 1:4] = torch.randn(4, 3, generator=torch.Generator().manual_seed(V)).to(dtype).cuda()
            index = torch.arange(1, 4).expand(4, 3).contiguous().cuda()
            teacher = torch.randn(4, 3).to(dtype).cuda()
            lse = torch.logsumexp(teacher.float(), 1) + 0.5
            check(z, index, teacher, lse, 1.0, torch.ones(4).cuda())
            _, grad = distillation_loss_grad(z, index, teacher, lse)
            assert (grad[:, 0] == 0).all() and (grad[:, 4:] == 0).all()
