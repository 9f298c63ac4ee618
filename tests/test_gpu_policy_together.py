"""GPU: the operators as they are used together - self-play into a move log, lambda returns of it, a cheap policy distilled from
the search's best moves, moves drafted with that policy, and the drafts verified against one batched search."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from tiny_net import TinyNet

pytestmark = pytest.mark.gpu


def test_self_play_returns_distillation_and_drafts():
    import bench
    from muzero_amd.drafts import verify_by_search
    from muzero_amd.mcts.mcts import MCTS
    from muzero_amd.network import MuZeroNetwork
    from muzero_amd.self_play import BatchedSelfPlay
    from muzero_amd.trainer import Trainer, distillation_loss
    cfg = bench.search_config(False, 2, 12, 1, 0.997)
    cfg.max_moves, cfg.dirichlet_alpha, cfg.exploration_frac = 12, 0.25, 0.25
    net = MuZeroNetwork(bench.cartpole_net_config(), seed=0)
    sp = BatchedSelfPlay(cfg, 'cartpole', net, 64, seed=0)
    log = sp.record(16)
    for _ in range(16):
        sp.step()
    returns = log.lambda_returns(0.997, 0.95)
    assert returns.shape == (16, 64) and returns.isfinite().all()
    ends = log.done[:16] != 0
    assert torch.equal(returns[ends], log.rewards[:16][ends])

    obs = log.observations[:16].reshape(-1, 1, 1, 4)
    teacher, index = torch.topk(torch.log(log.probs[:16].reshape(-1, 2).float()), 1, dim=1)   # the move the search prefers
    tcfg = SimpleNamespace(lr=0.05, lr_decay_rate=1.0, lr_decay_steps=1, weight_decay=0.0, momentum=0.9, support_limit=10,
                           value_loss_weight=1.0, optimizer='SGD')
    student = TinyNet(4, 2, 8, 10, seed=1).to('cuda')
    tr = Trainer(student, tcfg)
    policy = student.initial_inference(obs, False)[0]
    plain = torch.nn.functional.cross_entropy(policy, index[:, 0], reduction='none')
    loss = distillation_loss(policy, index, teacher)
    assert torch.allclose(loss, plain, rtol=1e-5, atol=1e-6)
    want = torch.autograd.grad(plain.mean(), student.pol.weight, retain_graph=True)[0]
    got = torch.autograd.grad(loss.mean(), student.pol.weight)[0]
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-6)
    assert np.isfinite(tr.distill(obs, index, teacher))

    B, K = 32, 3
    positions = log.observations[:K + 1, :B].transpose(0, 1).contiguous()          # [B, K + 1, 4]
    with torch.no_grad():
        draft = torch.softmax(student.initial_inference(positions[:, :K].reshape(-1, 1, 1, 4), False)[0].double(), 1).reshape(B, K, 2)
    tokens = (torch.rand(B, K, device='cuda') > draft[:, :, 0]).long()
    legal, to_play = np.ones((B, K + 1, 2)), np.zeros((B, K + 1), np.int64)
    search = lambda: verify_by_search(MCTS(cfg), net, positions.reshape(B, K + 1, 1, 1, 4), legal, to_play, tokens, draft, seed=5)  # noqa: E731
    np.random.seed(3)
    accepted, moves, values = search()
    assert accepted.shape == (B,) and moves.shape == (B, K + 1) and values.shape == (B, K + 1)
    # the same search and uniforms by hand, through the plain rule
    from test_gpu_drafts import plain as plain_rule
    np.random.seed(3)
    _, _, probs = MCTS(cfg).search_batch(net, positions.reshape(-1, 1, 1, 4), legal.reshape(-1, 2), to_play.reshape(-1), 1.0, seed=5)
    target = torch.as_tensor(np.asarray(probs)).reshape(B, K + 1, 2)
    ua, us = torch.as_tensor(np.random.random_sample((B, K))), torch.as_tensor(np.random.random_sample(B))
    n, want = plain_rule(tokens, draft, target, ua, us, None)
    np.testing.assert_array_equal(accepted.cpu().numpy(), n)
    np.testing.assert_array_equal(moves.cpu().numpy(), want)


def test_a_captured_training_step():
    """Forward and backward of the recurrence and the distillation in one graph, replayed over new inputs; the leaves belong to
    the capture alone (an eager graph of the same leaves must not live while a backward pass is captured)."""
    from muzero_amd.targets import linear_recurrence
    from muzero_amd.trainer import distillation_loss
    gen = torch.Generator().manual_seed(0)
    new = lambda *s: torch.randn(s, generator=gen).cuda()  # noqa: E731
    T, V = 900, 70                                          # a chain of links forward and backward, rows of two packs
    gate, x, dy = torch.sigmoid(new(1, T, V)), new(1, T, V), new(1, T, V)
    index = torch.randint(0, V, (T, 3), generator=gen).cuda()
    teacher, up = new(T, 3), torch.rand(T, generator=gen).cuda()

    def step(gate, x):
        y, _ = linear_recurrence(gate, x)
        loss = distillation_loss(y[0], index, teacher)
        return (loss,) + torch.autograd.grad(loss, (gate, x), up)

    leaves = lambda: (gate.clone().requires_grad_(), x.clone().requires_grad_())  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g, z = leaves()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(g, z)
    for i in range(4):
        with torch.no_grad():
            z.copy_(x * (1 + i))
        graph.replay()
        want = step(gate.clone().requires_grad_(), (x * (1 + i)).requires_grad_())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
