"""GPU: calls of more rows than one launch can take (a grid has fewer than 2^32 threads), which run in slices: what stands on both
sides of every slice's border is right, and what a call of these rows alone gives."""
import pytest
import torch

from test_gpu_recurrence import close, inputs, loop, loop_backward

pytestmark = pytest.mark.gpu
SLICE = 1 << 20


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize('B,T,D,layout', [(2 * SLICE + 5, 9, 1, 'rows'), (3, 9, SLICE // 2 + 7, 'rows'), (2, 10, 2 * SLICE + 3, 'rows'),
                                          (SLICE + 3, 9, 2, 'channels'), (SLICE // 2 + 3, 9, 70, 'channels'), (2, 9, 64 * SLICE + 35, 'channels'),
                                          (SLICE + 1, 3, 1, 'rows'), (2 * SLICE + 1, 2, 3, 'channels')])
def test_recurrence(B, T, D, layout, dtype):
    from muzero_amd.targets import linear_recurrence
    if B * T * D > 1 << 29 and dtype != torch.bfloat16:
        pytest.skip('the slices of channels are those of the smallest type')
    # some sequences and channels at each border, made on their own; all others hold one record over and over
    marks = sorted({b for at in (0, SLICE // max(D, 1), SLICE // max((D + 63) // 64, 1), SLICE // max((D + 31) // 32, 1), SLICE, 2 * SLICE, B // 2, B)
                    for b in range(at - 2, at + 2) if 0 <= b < B})
    chans = sorted({d for at in (0, SLICE, 2 * SLICE, 32 * SLICE, 64 * SLICE, D) for d in range(at - 3, at + 3) if 0 <= d < D})
    a1, x1, s1 = inputs(1, T, 1, dtype, seed=T)
    shape = (B, T, D) if layout == 'channels' else (B, D, T)
    turn = (lambda t: t) if layout == 'channels' else (lambda t: t.transpose(1, 2))
    make = lambda: turn(torch.empty(shape, dtype=dtype, device='cuda'))  # noqa: E731
    a, x = make().copy_(a1.expand(B, T, D)), make().copy_(x1.expand(B, T, D))
    s = s1.expand(B, D).contiguous()
    bi, di = torch.tensor(marks).cuda()[:, None, None], torch.tensor(chans).cuda()[None, None, :]
    n, m = len(marks), len(chans)
    ac, xc, sc = inputs(n, T, m, dtype, seed=T + 1)
    ti = torch.arange(T).cuda()[None, :, None]
    a[bi, ti, di], x[bi, ti, di], s[bi[:, 0], di[:, 0]] = ac, xc, sc
    leaves = [t.requires_grad_() for t in (a, x, s)]
    y, last = linear_recurrence(*leaves)
    y_ref, last_ref = loop(ac, xc, sc, False)
    z, zl = loop(ac.abs(), xc.abs(), sc.abs(), False)
    close(y.detach()[bi, ti, di], y_ref, z, T, dtype)
    close(last.detach()[bi[:, 0], di[:, 0]], last_ref, zl, T, dtype)
    dy = x.detach()
    da, dx, ds = torch.autograd.grad(y, leaves, dy)
    dx_ref, da_ref, ds_ref = loop_backward(ac, y_ref, sc, xc, None, False)
    zx, zda, zs = loop_backward(ac.abs(), z, sc.abs(), xc.abs(), None, False)
    close(dx[bi, ti, di], dx_ref, zx, T, dtype)
    close(da[bi, ti, di], da_ref, 2 * zda, T, dtype)
    close(ds[bi[:, 0], di[:, 0]], ds_ref, zs, T + 1, dtype)
    # every other row and channel holds the same record
    rest = torch.ones(B, dtype=torch.bool, device='cuda')
    rest[bi[:, 0, 0]] = False
    if rest.any():
        only = y.detach()[rest]
        assert (only == only[:1]).all()


@pytest.mark.parametrize('V', [9, 40, 70])
def test_distillation(V):
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    R = 2 * SLICE + 3
    g = torch.Generator(device='cuda').manual_seed(V)
    z = torch.randn(R, V, generator=g, device='cuda').bfloat16()
    index = torch.randint(-1, V, (R, 3), generator=g, device='cuda', dtype=torch.int32)
    teacher, weight = torch.randn(R, 3, generator=g, device='cuda'), torch.rand(R, generator=g, device='cuda')
    lse = torch.logsumexp(teacher, 1) + 0.3
    loss, grad = distillation_loss_grad(z, index, teacher, lse, 1.0, weight)
    leaf = z.requires_grad_()
    loss2 = distillation_loss(leaf, index, teacher, lse, 1.0, weight)
    up = torch.rand(R, generator=g, device='cuda')
    grad2, = torch.autograd.grad(loss2, leaf, up)
    for at in (0, SLICE, 2 * SLICE):
        part = slice(max(at - 3, 0), at + 3)
        one, done = distillation_loss_grad(z.detach()[part], index[part], teacher[part], lse[part], 1.0, weight[part])
        few = z.detach()[part].requires_grad_()
        total = distillation_loss(few, index[part], teacher[part], lse[part], 1.0, weight[part])
        assert torch.equal(loss[part], one) and torch.equal(grad[part], done) and torch.equal(loss2[part], total)
        assert torch.equal(grad2[part], torch.autograd.grad(total, few, up[part])[0])


def test_more_rows_than_threads_of_a_grid():
    """2^26 rows of a wave each: 2^32 threads."""
    from muzero_amd.drafts import verify_drafts
    from muzero_amd.targets import linear_recurrence
    from muzero_amd.trainer import distillation_loss
    n = (1 << 26) + 3
    x = torch.ones(n, 2, 2, dtype=torch.bfloat16, device='cuda').transpose(1, 2)     # time contiguous
    y, last = linear_recurrence(x[:, :, :1], x[:, :, :1])
    assert (y[:, 0] == 1).all() and (y[:, 1] == 2).all() and (last == 2).all()
    y, last = linear_recurrence(x, x)
    assert (y[:, 0] == 1).all() and (y[:, 1] == 2).all() and (last == 2).all()
    z = torch.zeros(1, 65, dtype=torch.bfloat16, device='cuda').expand(n, 65)
    loss = distillation_loss(z, torch.zeros(1, 1, dtype=torch.int32, device='cuda').expand(n, 1), torch.zeros(1, 1, device='cuda').expand(n, 1))
    assert (loss == loss[0]).all() and abs(float(loss[0]) - 4.1743872699) < 1e-5     # log 65
    target = torch.full((1, 1, 65), 1.0, dtype=torch.bfloat16, device='cuda').expand(n, 1, 65)
    u = torch.linspace(0, 0.999, n, dtype=torch.float64, device='cuda')
    accepted, out = verify_drafts(torch.zeros(n, 0, dtype=torch.int32, device='cuda'), None, target, torch.zeros(n, 0, dtype=torch.float64, device='cuda'), u)
    assert (accepted == 0).all() and torch.equal(out[:, 0], (u * 65).int())


@pytest.mark.parametrize('V', [9, 70, 300])
def test_verification(V):
    from muzero_amd.drafts import verify_drafts
    B, K = SLICE + 5, 2
    g = torch.Generator(device='cuda').manual_seed(V)
    target = torch.rand(B, K + 1, V, generator=g, device='cuda').bfloat16()
    draft = torch.rand(B, K, V, generator=g, device='cuda').bfloat16()
    tokens = torch.randint(0, V, (B, K), generator=g, device='cuda')
    ua, us = (torch.rand(s, generator=g, device='cuda', dtype=torch.float64) for s in ((B, K), (B,)))
    lengths = torch.randint(0, K + 1, (B,), generator=g, device='cuda', dtype=torch.int32)
    for d in (draft, None):
        n, out = verify_drafts(tokens, d, target, ua, us, lengths)
        part = slice(SLICE - 4, B)
        n1, out1 = verify_drafts(tokens[part], None if d is None else d[part], target[part], ua[part], us[part], lengths[part])
        assert torch.equal(n[part], n1) and torch.equal(out[part], out1)
        n0, out0 = verify_drafts(tokens[:5], None if d is None else d[:5], target[:5], ua[:5], us[:5], lengths[:5])
        assert torch.equal(n[:5], n0) and torch.equal(out[:5], out0)
