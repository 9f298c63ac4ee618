"""GPU: distillation from a teacher's top logits (mz_distill_loss, mz_distill_grad, mz_distill_loss_grad) against the definition
in float64 under autograd: actions from one to a wide odd set, entries absent, repeated or at -inf, rows that count for
nothing, masked logits, strides, types, captured graphs, and the trainer's use of it.

Tolerance: exp2's argument carries |t| + 1 roundings of 2^-24 and the exponential two more units, so a term of the softmax sum
is off by at most (|t| + 4) 2^-23 of itself and the sum by the average of that plus its additions (at most V / 64 + 16 a
thread): `rel` below.  The loss takes the logarithm of one or two such sums, a gradient entry one quotient, then one rounding
to its type."""
import math
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def definition(logits, index, teacher, lse, tau, weight):
    """(loss, d loss / d logits, tolerances of both), float64 on the host."""
    z = logits.detach().double().cpu().requires_grad_()
    index, t = index.long().cpu(), teacher.double().cpu() / tau
    R, V = z.shape
    there = (index >= 0) & (index < V)
    at = torch.where(there, index, 0)
    t = torch.where(there, t, -math.inf)
    w = torch.ones(R, dtype=torch.float64) if weight is None else weight.double().cpu()
    loss, p_row, rests, qrests = [], torch.zeros(R, V, dtype=torch.float64), torch.zeros(R), torch.ones(R)
    for r in range(R):
        if w[r] == 0 or not there[r].any():
            loss.append((z[r] * 0).nan_to_num(0, 0, 0).sum() * 0)
            continue
        logq = torch.log_softmax(z[r] / tau, 0)
        if lse is None:
            p = torch.softmax(t[r], 0) if (t[r] > -math.inf).any() else torch.zeros_like(t[r])
        else:
            p = torch.exp(t[r] - lse[r].double().cpu())
        logp = torch.log(p)
        kl = sum((p[k] * (logp[k] - logq[at[r, k]]) for k in range(len(p)) if p[k] > 0), torch.zeros((), dtype=torch.float64))
        inside = torch.zeros(V, dtype=torch.bool)
        inside[at[r][there[r]]] = True
        p_row[r].index_add_(0, at[r], p)
        if lse is not None and not inside.all():
            rest = (1 - p.sum()).clamp(min=0)
            logrest = torch.logsumexp(logq[~inside], 0)
            if rest > 0 and logrest > -math.inf:
                kl = kl + rest * (torch.log(rest) - logrest)
                rests[r], qrests[r] = rest, torch.exp(logrest.detach())
        loss.append(w[r] * tau * tau * kl)
    loss = torch.stack(loss)
    grad, = torch.autograd.grad(loss.sum(), z)
    with torch.no_grad():
        q = torch.softmax(z / tau, 1).nan_to_num(0)
        steps = ((z.max(1, keepdim=True).values - z) / tau * math.log2(math.e)).nan_to_num(0, 0, 0).clamp(max=200)
        rel = ((q * steps).sum(1) + 16 + V / 64) * 2.0 ** -23
        mass = p_row.sum(1) + rests
        tol_loss = (w * tau * tau).abs() * (mass + 2 * rests) * rel
        tol_grad = (w * tau).abs()[:, None] * q * ((rel[:, None] + (steps + 4) * 2.0 ** -23) * (mass + 2 * rests / qrests)[:, None])
    return loss.detach(), torch.where((w != 0)[:, None], grad, 0.0), tol_loss, tol_grad


def check(logits, index, teacher, lse, tau, weight):
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    want, dwant, tol, dtol = definition(logits, index, teacher, lse, tau, weight)
    loss, grad = distillation_loss_grad(logits, index, teacher, lse, tau, weight)
    leaf = logits.detach().requires_grad_()
    loss2 = distillation_loss(leaf, index, teacher, lse, tau, weight)
    up = torch.linspace(0.5, -2.0, len(loss), device='cuda')
    grad2, = torch.autograd.grad(loss2, leaf, up)
    half = torch.finfo(logits.dtype).eps / 2
    least = 2.0 ** -25 if logits.dtype == torch.float16 else 1e-37
    for got in (loss, loss2):
        assert got.dtype == torch.float32 and got.shape == want.shape
        got = got.double().cpu()
        same = (got == want) | ((got - want).abs() <= tol + 2.0 ** -23 * want.abs())
        assert same.all(), ((got - want).abs() / (tol + 1e-30)).max()
    for got, ref, dt in ((grad, dwant, dtol), (grad2, dwant * up.double().cpu()[:, None], dtol * up.double().cpu().abs()[:, None])):
        assert got.dtype == logits.dtype and got.shape == logits.shape
        off = (got.double().cpu() - ref).abs()
        allowed = dt * (1 + half) + (half + 2.0 ** -23) * ref.abs() + least
        assert (off <= allowed).all(), ((off / allowed).max(), (off > allowed).nonzero()[:3])
    return loss, grad


def rows(R, V, K, dtype, seed, tau, tail, pad=True, index_type=torch.int64):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(R, V, generator=g) * 3
    teacher = logits + torch.randn(R, V, generator=g)
    top, index = torch.topk(teacher, K, dim=1)
    lse = torch.logsumexp(teacher / tau, 1) if tail else None
    weight = torch.where(torch.rand(R, generator=g) < 0.2, torch.zeros(()), torch.rand(R, generator=g) + 0.5)
    if pad:
        index = torch.where(torch.rand(R, K, generator=g) < 0.2, -1, index)
    return (logits.to(dtype).cuda(), index.to(index_type).cuda(), top.to(dtype).cuda(), None if lse is None else lse.float().cuda(),
            weight.cuda())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('R,V,K', [(1, 1, 1), (5, 2, 1), (33, 9, 4), (3, 9, 9), (2, 64, 64), (6, 65, 3), (3, 255, 17), (2, 1000, 100),
                                   (2, 2049, 5), (3, 4099, 70), (2, 8200, 2), (1, 16390, 33), (2, 33001, 16), (1, 70001, 130)])
def test_loss_and_gradient(R, V, K, dtype):
    for tau, tail in ((1.0, False), (2.5, True)):
        logits, index, teacher, lse, weight = rows(R, V, K, dtype, V + K, tau, tail, index_type=torch.int32 if tail else torch.int64)
        check(logits, index, teacher, lse, tau, weight)
        check(logits, index, teacher, lse, tau, None)


def test_a_wide_odd_row_in_every_type():
    for dtype in TYPES:
        logits, index, teacher, lse, weight = rows(1, 131071, 64, dtype, 5, 2.0, True, pad=False)
        check(logits, index, teacher, lse, 2.0, None)


@pytest.mark.parametrize('V', [6, 300, 5000])
def test_entries_named_twice_absent_and_impossible(V):
    index = torch.tensor([[0, 0, 0, 1], [2, 5, 2, 5], [-1, -1, -1, -1], [V, -7, 3, V + 10], [4, 4, -1, 4], [1, 2, 3, 4]]).cuda()
    teacher = torch.tensor([[0.5, 1.0, -1.0, 0.0], [2.0, -math.inf, 1.0, 0.3], [1.0, 2.0, 3.0, 4.0], [9.0, math.nan, 1.0, math.inf],
                            [1.0, 1.0, math.nan, 0.0], [-math.inf] * 4]).cuda()
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(6, V, generator=g).cuda()
    loss, grad = check(logits, index, teacher, None, 1.0, None)
    assert loss[2] == 0 and (grad[2] == 0).all() and loss[5] == 0 and (grad[5] == 0).all()
    check(logits.half(), index, teacher, torch.full((6,), 4.0).cuda(), 1.5, None)


def test_rows_of_no_weight_hold_anything():
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    for V in (9, 700, 20001):
        logits, index, teacher, _, _ = rows(4, V, 3, torch.float32, 2, 1.0, False, pad=False)
        weight = torch.tensor([0.0, 1.0, 0.0, 2.0]).cuda()
        clean, cgrad = distillation_loss_grad(logits, index, teacher, weight=weight)
        logits[0], logits[2], teacher[2] = math.nan, -math.inf, math.nan
        loss, grad = distillation_loss_grad(logits, index, teacher, weight=weight)
        assert torch.equal(loss, clean) and torch.equal(grad, cgrad) and (grad[0] == 0).all() and loss[0] == 0
        leaf = logits.requires_grad_()
        total = distillation_loss(leaf, index, teacher, weight=weight)
        g, = torch.autograd.grad(total.sum(), leaf)
        assert g.isfinite().all() and (g[0] == 0).all() and (g[2] == 0).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V,K', [(1, 70), (3, 100), (5, 1024), (300, 300), (17, 65), (2041, 66), (1009, 70)])
def test_more_entries_than_lanes(V, K, dtype):
    """Long lists of entries, most actions named several times, rows that begin anywhere in a pack of 16 bytes."""
    g = torch.Generator().manual_seed(K)
    logits = (torch.randn(7, V, generator=g) * 2).to(dtype).cuda()
    index = torch.randint(-1, V + 1, (7, K), generator=g).int().cuda()
    teacher = torch.randn(7, K, generator=g).to(dtype).cuda()
    check(logits, index, teacher, None, 1.0, None)
    check(logits, index, teacher, torch.full((7,), math.log(K) + 2.0).cuda(), 0.7, None)


@pytest.mark.parametrize('V', [9, 500, 9000])
def test_masked_logits(V):
    """Illegal actions at -inf or at the type's lowest value take no part; a teacher that names one gives an infinite loss."""
    from muzero_amd.trainer import distillation_loss_grad
    logits, index, teacher, _, _ = rows(3, V, 2, torch.float32, 4, 1.0, False, pad=False)
    legal = torch.zeros(3, V, dtype=torch.bool).cuda()
    legal[:, :5] = True
    index = torch.tensor([[0, 4], [1, 2], [3, 0]]).cuda()
    for low in (-math.inf, torch.finfo(torch.float32).min):
        z = torch.where(legal, logits, low)
        loss, grad = distillation_loss_grad(z, index, teacher)
        few, fgrad = distillation_loss_grad(z[:, :5].contiguous(), index, teacher)
        assert torch.allclose(loss, few, rtol=1e-6) and torch.allclose(grad[:, :5], fgrad, rtol=1e-5, atol=1e-7)
        assert (grad[:, 5:] == 0).all()
        # every legal action named and the rest of the mass known: nothing is left outside, whatever rounding says
        every = torch.arange(5).expand(3, 5).contiguous().cuda()
        top = torch.randn(3, 5).cuda()
        kl, kgrad = distillation_loss_grad(z, every, top, teacher_lse=torch.logsumexp(top, 1) + 1e-6)
        assert kl.isfinite().all() and kgrad.isfinite().all()
    outside = torch.tensor([[0, V - 1]] * 3).cuda()
    loss, grad = distillation_loss_grad(torch.where(legal, logits, -math.inf), outside, teacher)
    assert (loss == math.inf).all() and grad.isfinite().all()
    loss, grad = distillation_loss_grad(torch.full((1, V), -math.inf).cuda(), index[:1], teacher[:1])
    assert loss.isnan().all()


def test_strides_and_neighbours():
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    for dtype in TYPES:
        for V in (9, 1001, 9999):
            logits, index, teacher, _, weight = rows(5, V, 4, dtype, 8, 1.0, False)
            room = torch.full((5, V + 6), math.nan, dtype=dtype, device='cuda')
            part = room[:, 3:-3]
            part.copy_(logits)
            want = distillation_loss_grad(logits, index, teacher, weight=weight)
            check(part, index, teacher, None, 1.0, weight)
            by_column = logits.t().contiguous().t()
            got = distillation_loss_grad(by_column, index.t().contiguous().t(), teacher, weight=weight)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            one = distillation_loss(logits[:1].expand(5, V), index, teacher, weight=weight)
            assert torch.equal(one[0], want[0][0])


def test_captured_and_replayed():
    from muzero_amd.trainer import distillation_loss_grad
    for R, V, K in ((40, 9, 4), (6, 33000, 20)):
        logits, index, teacher, lse, weight = rows(R, V, K, torch.bfloat16, 6, 1.0, True)
        z = logits.clone()
        distillation_loss_grad(z, index, teacher, lse, 1.0, weight)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss, grad = distillation_loss_grad(z, index, teacher, lse, 1.0, weight)
        for i in range(4):
            z.copy_(logits * (0.5 + i))
            graph.replay()
            want = distillation_loss_grad(logits * (0.5 + i), index, teacher, lse, 1.0, weight)
            torch.cuda.synchronize()
            assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])


def test_trainer_distils_the_policy():
    """The gradient that reaches the network is the one plain torch operations give for the same loss."""
    from tiny_net import TinyNet
    from muzero_amd.trainer import Trainer
    cfg = SimpleNamespace(lr=0.05, lr_decay_rate=1.0, lr_decay_steps=1, weight_decay=0.0, momentum=0.0, support_limit=5,
                          value_loss_weight=1.0, optimizer='SGD')
    net = TinyNet(4, 6, 8, 5, seed=0).to('cuda')
    g = torch.Generator().manual_seed(0)
    obs = torch.randn(32, 1, 1, 4, generator=g).cuda()
    teacher, index = torch.topk(torch.randn(32, 6, generator=g).cuda() * 2, 3, dim=1)
    policy = net.initial_inference(obs, False)[0]
    p = torch.softmax(teacher, 1)
    plain = (p * (torch.log(p) - torch.log_softmax(policy, 1).gather(1, index))).sum(1).mean()
    want = torch.autograd.grad(plain, [w for w in net.parameters()], allow_unused=True)
    before = [w.detach().clone() for w in net.parameters()]
    tr = Trainer(net, cfg)
    loss = tr.distill(obs, index, teacher)
    assert abs(loss - float(plain.detach())) <= 1e-5 * abs(float(plain.detach())) + 1e-6 and tr.training_step == 1
    for w, b, grad in zip(net.parameters(), before, want):
        step = torch.zeros_like(b) if grad is None else cfg.lr * grad
        assert torch.allclose(w, b - step, rtol=1e-5, atol=1e-6)


def test_offsets_beyond_32_bits():
    """Rows whose distance in memory passes 2^31 elements."""
    from muzero_amd.trainer import distillation_loss_grad
    big = 2 ** 31 + 16
    room = torch.empty(big + 200000, dtype=torch.bfloat16, device='cuda')
    for V in (9, 700, 5000, 140000):
        logits, index, teacher, _, _ = rows(2, V, 3, torch.bfloat16, V, 1.0, False, pad=False)
        far = room.as_strided((2, V), (big, 1), 5)
        far.copy_(logits)
        loss, grad = distillation_loss_grad(far, index, teacher)
        want = distillation_loss_grad(logits, index, teacher)
        assert torch.allclose(loss, want[0], rtol=1e-5, atol=1e-6) and torch.allclose(grad, want[1], rtol=2.0 ** -7, atol=1e-9)


def test_not_a_number_shows():
    """A NaN logit makes its row NaN, whatever stands before it, and no other row."""
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    for V in (9, 100, 800, 5000, 60000):
        for at, low in ((0, False), (V - 1, False), (V // 2, True)):
            logits, index, teacher, lse, _ = rows(3, V, 2, torch.bfloat16, V, 1.0, True, pad=False)
            if low:
                logits[1, :V // 2] = -math.inf
            index[1] = torch.tensor([V - 2, V - 1])
            logits[1, at] = math.nan
            for tail in (lse, None):
                leaf = logits.detach().requires_grad_()
                total = distillation_loss(leaf, index, teacher, tail)
                g, = torch.autograd.grad(total.sum(), leaf)
                loss, grad = distillation_loss_grad(logits, index, teacher, tail)
                for lo, gr in ((total, g), (loss, grad)):
                    assert lo[1].isnan() and gr[1].isnan().all() and lo[[0, 2]].isfinite().all() and gr[[0, 2]].isfinite().all()


def test_refusals():
    from muzero_amd.engine import EngineError
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    z, i, t = torch.zeros(4, 9, device='cuda'), torch.zeros(4, 2, dtype=torch.int64, device='cuda'), torch.zeros(4, 2, device='cuda')
    f = torch.zeros(4, device='cuda')
    for call in (distillation_loss, distillation_loss_grad):
        for args in ((z[0], i, t), (z, i[0], t), (z, i[:3], t), (z, i, t[:, :1]), (z.double(), i, t), (z, i, t.double()), (z, i.short(), t),
                     (z, i, t, f.double()), (z, i, t, f[:3]), (z, i, t, None, 1.0, f[:2]), (z, i, t, None, 0.0), (z, i, t, None, math.nan),
                     (z, i[:, :0], t[:, :0]), (z, i.expand(2, 4, 2)[0].repeat(1, 600), t.repeat(1, 600))):
            with pytest.raises(ValueError, match='distill'):
                call(*args)
        with pytest.raises(EngineError, match='device tensors'):
            call(z, i.cpu(), t)
        assert call(z[:0], i[:0], t[:0])[0].shape[0] == 0 if call is distillation_loss_grad else call(z[:0], i[:0], t[:0]).shape == (0,)
    leaf = z.clone().requires_grad_()
    g, = torch.autograd.grad(distillation_loss(leaf, i, t).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)


def test_two_streams_at_once():
    from muzero_amd.trainer import distillation_loss_grad
    args = [rows(300, 5000, 20, torch.bfloat16, s, 1.0, False)[:3] for s in (1, 2)]
    want = [distillation_loss_grad(*a) for a in args]
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for st, a in zip(streams, args):
            with torch.cuda.stream(st):
                got.append(distillation_loss_grad(*a))
    torch.cuda.synchronize()
    assert all(torch.equal(g[0], want[k % 2][0]) and torch.equal(g[1], want[k % 2][1]) for k, g in enumerate(got))
