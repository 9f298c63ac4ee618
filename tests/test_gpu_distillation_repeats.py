"""GPU: rows that name an action more than once.  Every entry has its own term, so the loss is the divergence of the summed
probabilities less the entropy of the choice between the entries of one action; the gradient is that of the merged row.

Tolerance: the loss's and gradient's own (test_gpu_distillation: `rel` at most (|t| + 16 + V / 64) 2^-23 with |t| < 16 here),
2^-17 in all with the merged row's."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_two_equal_entries_alone():
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    z = torch.zeros(1, 1, device='cuda')
    index, teacher = torch.zeros(1, 2, dtype=torch.int64, device='cuda'), torch.zeros(1, 2, device='cuda')
    for loss in (distillation_loss(z, index, teacher), distillation_loss_grad(z, index, teacher)[0]):
        assert abs(float(loss) + math.log(2)) <= 2.0 ** -23
    loss, grad = distillation_loss_grad(z, index[:, :1], teacher[:, :1])
    assert float(loss) == 0 and float(grad) == 0


@pytest.mark.parametrize('V,K', [(5, 8), (50, 30), (600, 64), (600, 200), (9001, 20)])
@pytest.mark.parametrize('tail', [False, True])
def test_against_the_merged_row(V, K, tail):
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    g = torch.Generator().manual_seed(V + K)
    R = 5
    z = torch.randn(R, V, generator=g).cuda()
    half = torch.stack([torch.randperm(V, generator=g)[:K // 2] for _ in range(R)])
    index, teacher = torch.cat([half, half], 1).cuda(), torch.randn(R, K // 2 * 2, generator=g).cuda()   # every action twice
    lse = torch.logsumexp(teacher, 1) + 0.5 if tail else None
    merged = torch.logsumexp(torch.stack(teacher.double().chunk(2, 1)), 0)
    p = torch.softmax(teacher.double(), 1) * (math.exp(-0.5) if tail else 1.0)
    choice = (p * (torch.cat([merged, merged], 1) - teacher.double())).sum(1)
    want, dwant = distillation_loss_grad(z, half.cuda(), merged.float(), teacher_lse=lse)
    leaf = z.clone().requires_grad_()
    loss2 = distillation_loss(leaf, index, teacher, teacher_lse=lse)
    grad2, = torch.autograd.grad(loss2.sum(), leaf)
    loss, grad = distillation_loss_grad(z, index, teacher, teacher_lse=lse)
    for got in (loss, loss2.detach()):
        assert ((got.double() - (want.double() - choice)).abs() <= 2.0 ** -17 * (1 + choice.abs())).all()
    for got in (grad, grad2):
        assert ((got - dwant).abs() <= 2.0 ** -17 * (1 + dwant.abs())).all()
