"""GPU: verification of drafted moves (mz_verify_drafts) against a plain float64 loop, value for value: every type, actions from
one to a wide odd set, ragged and empty drafts, drafts without probabilities, rows that leave nothing, entries that are no
probabilities, strides, captured graphs - and the moves that come out are distributed as the target's."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


def plain(tokens, draft, target, ua, us, lengths):
    clean = lambda v: np.where((v > 0) & np.isfinite(v), v, 0.0)  # noqa: E731
    tokens, target = tokens.cpu().numpy(), clean(target.double().cpu().numpy())
    draft = None if draft is None else clean(draft.double().cpu().numpy())
    ua, us = ua.cpu().numpy(), us.cpu().numpy()
    B, K = tokens.shape
    V = target.shape[2]
    n_out, out = np.zeros(B, np.int32), np.full((B, K + 1), -1, tokens.dtype)
    for b in range(B):
        length = K if lengths is None else int(np.clip(int(lengths[b]), 0, K))
        n = 0
        while n < length:
            x = tokens[b, n]
            if not (0 <= x < V and ua[b, n] * (1.0 if draft is None else draft[b, n, x]) < target[b, n, x]):
                break
            n += 1
        row = target[b, n]
        if n < length:
            less = row.copy()
            if draft is None:
                if 0 <= tokens[b, n] < V:
                    less[tokens[b, n]] = 0.0
            else:
                less = np.maximum(row - draft[b, n], 0.0)
            row = less if less.max() > 0 else row
        sums = np.cumsum(row)
        over = np.nonzero((sums > us[b] * sums[-1]) & (row > 0))[0]
        some = np.nonzero(row > 0)[0]
        out[b, :n] = tokens[b, :n]
        out[b, n] = over[0] if len(over) else some[-1] if len(some) else -1
        n_out[b] = n
    return n_out, out


def case(B, K, V, dtype, seed, token_type=torch.int64, noise=0.7):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, K + 1, V, generator=g, dtype=torch.float64) * 2
    target = torch.softmax(z, 2)
    draft = torch.softmax(z[:, :K] + noise * torch.randn(B, K, V, generator=g, dtype=torch.float64), 2)
    tokens = torch.multinomial(draft.reshape(B * K, V), 1, generator=g).reshape(B, K) if K else torch.zeros(B, 0, dtype=torch.int64)
    u = lambda *s: torch.rand(s, generator=g, dtype=torch.float64).cuda()  # noqa: E731
    return tokens.to(token_type).cuda(), draft.to(dtype).cuda(), target.to(dtype).cuda(), u(B, K), u(B)


def check(tokens, draft, target, ua, us, lengths=None):
    from muzero_amd.drafts import verify_drafts
    n, out = verify_drafts(tokens, draft, target, ua, us, lengths=lengths)
    want_n, want = plain(tokens, draft, target, ua, us, None if lengths is None else lengths.cpu().numpy())
    assert n.dtype == torch.int32 and out.dtype == tokens.dtype
    np.testing.assert_array_equal(n.cpu().numpy(), want_n)
    np.testing.assert_array_equal(out.cpu().numpy(), want)
    return n, out


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,K,V', [(1, 1, 1), (7, 0, 5), (33, 5, 9), (300, 3, 2), (5, 4, 64), (5, 4, 65), (4, 12, 129), (6, 2, 1000), (3, 7, 1025),
                                   (2, 3, 8193), (1, 4, 32000), (3, 2, 50021), (1, 70, 300), (1, 2, 131071)])
def test_against_the_plain_loop(B, K, V, dtype):
    for seed, token_type in ((0, torch.int64), (1, torch.int32)):
        tokens, draft, target, ua, us = case(B, K, V, dtype, seed, token_type)
        check(tokens, draft, target, ua, us)
        check(tokens, None, target, ua, us)
        lengths = torch.randint(-1, K + 2, (B,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()
        check(tokens, draft, target, ua, us, lengths)


@pytest.mark.parametrize('V', [3, 70, 5000, 40000])
def test_rows_that_leave_little_or_nothing(V):
    B = 8
    tokens, draft, target, ua, us = case(B, 2, V, torch.float32, 3)
    target[0] = 0.0                                             # no mass anywhere: no token
    target[1, 0] = draft[1, 0] * 0.5                            # nowhere above the draft: the target's own row
    ua[1, 0] = 0.9
    target[2, 0], draft[2, 0] = draft[2, 0].clone(), draft[2, 0].clone()   # equal rows: every draft is kept
    target[3, 0] = 0.0
    target[3, 0, V - 1] = 1.0                                   # one action only, the last
    target[4, 0], target[4, 0, :2] = -1.0, float('nan')         # no probabilities at all
    target[5, 0, V // 2], draft[5, 0, 0] = float('inf'), float('nan')
    tokens[6, 0], tokens[6, 1] = V, 0                           # outside the actions
    tokens[7, 0] = -1
    us[3], us[2] = 1.0 - 2.0 ** -53, 0.0
    n, out = check(tokens, draft, target, ua, us)
    assert n[0] == 0 and out[0, 0] == -1 and n[6] == 0 and n[7] == 0
    check(tokens, None, target, ua, us)
    for u in (0.0, 1.0 - 2.0 ** -53, 0.5):
        check(tokens, draft, target, ua, torch.full((B,), u, dtype=torch.float64).cuda())


def test_dyadic_ties_go_past_the_border():
    """Running sums that equal u times the whole exactly: the index behind them is taken, as searchsorted(side='right')."""
    for V in (4, 128, 4096):
        target = torch.full((V, 1, V), 1.0 / V).cuda()
        us = (torch.arange(V, dtype=torch.float64) / V).cuda()
        tokens = torch.zeros(V, 0, dtype=torch.int32).cuda()
        _, out = check(tokens, None, target, torch.zeros(V, 0, dtype=torch.float64).cuda(), us)
        assert torch.equal(out[:, 0].cpu(), torch.arange(V, dtype=torch.int32))


def test_strides():
    tokens, draft, target, ua, us = case(4, 3, 77, torch.bfloat16, 5)
    room = torch.zeros(4, 9, 80, dtype=torch.bfloat16).cuda()
    room[:, 1:8:2, 2:79] = target
    part = room[:, 1:8:2, 2:79]
    want = check(tokens, draft, target, ua, us)
    for t, d in ((part, draft), (target.transpose(0, 1).contiguous().transpose(0, 1), draft.transpose(1, 2).contiguous().transpose(1, 2))):
        got = check(tokens.t().contiguous().t(), d, t, ua, us)
        assert torch.equal(got[1], want[1])
    same = target[:, :1].expand(4, 4, 77)
    check(tokens, same[:, :3], same, ua, us)


def test_moves_are_distributed_as_the_target():
    """40000 independent pairs over 6 actions: the first move's counts lie within 5 standard deviations of the target's."""
    n = 40000
    g = torch.Generator().manual_seed(0)
    target = torch.softmax(torch.randn(6, generator=g), 0)
    draft = torch.softmax(torch.randn(6, generator=g), 0)
    tokens = torch.multinomial(draft, n, replacement=True, generator=g)[:, None].cuda()
    from muzero_amd.drafts import verify_drafts
    u = torch.rand(n, 2, generator=g, dtype=torch.float64).cuda()
    _, out = verify_drafts(tokens, draft.expand(n, 1, 6).cuda(), target.expand(n, 2, 6).cuda(), u[:, :1], u[:, 1])
    counts = torch.bincount(out[:, 0].cpu(), minlength=6).double()
    assert ((counts - n * target.double()).abs() <= 5 * (n * target.double() * (1 - target.double())).sqrt()).all()


def test_captured_and_replayed():
    from muzero_amd.drafts import verify_drafts
    for B, K, V in ((30, 3, 9), (2, 4, 40000)):
        tokens, draft, target, ua, us = case(B, K, V, torch.float32, 7)
        verify_drafts(tokens, draft, target, ua, us)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            n, out = verify_drafts(tokens, draft, target, ua, us)
        for i in range(4):
            ua.copy_(torch.rand(B, K, dtype=torch.float64))
            us.copy_(torch.rand(B, dtype=torch.float64))
            graph.replay()
            want = verify_drafts(tokens, draft, target, ua, us)
            torch.cuda.synchronize()
            assert torch.equal(n, want[0]) and torch.equal(out, want[1])


def test_offsets_beyond_32_bits():
    big = 2 ** 31 + 8
    room = torch.empty(2 * big + 300000, dtype=torch.bfloat16, device='cuda')
    for V in (9, 100, 70000):
        tokens, draft, target, ua, us = case(2, 1, V, torch.bfloat16, 4)
        for strides in ((big, V, 1), (V, big, 1)):
            far = room.as_strided((2, 2, V), strides, 3)
            far.copy_(target)
            check(tokens, draft, far, ua, us)
            check(tokens, far[:, :1], target, ua, us)


def test_refusals():
    from muzero_amd.drafts import verify_drafts
    from muzero_amd.engine import EngineError
    tokens, draft, target, ua, us = case(3, 2, 9, torch.float32, 0)
    n = torch.zeros(3, dtype=torch.int32).cuda()
    for args in ((tokens[0], draft, target, ua, us), (tokens, draft[:, :1], target, ua, us), (tokens, draft, target[:, :2], ua, us),
                 (tokens, draft.double(), target, ua, us), (tokens.float(), draft, target, ua, us), (tokens, draft, target, ua.float(), us),
                 (tokens, draft, target, ua, us[:2]), (tokens, draft, target.int(), ua, us), (tokens, draft, target, ua, us, n.long()),
                 (tokens, draft, target, ua, us, n[:2]), (tokens, draft[:, :, :0], target[:, :, :0], ua, us)):
        with pytest.raises(ValueError, match='verify_drafts'):
            verify_drafts(*args)
    with pytest.raises(EngineError, match='device tensors'):
        verify_drafts(tokens, draft.cpu(), target, ua, us)
    wide = torch.zeros(1, 1, 1, dtype=torch.float16).cuda().expand(1, 1, (1 << 20) + 1)
    with pytest.raises(ValueError, match='actions'):
        verify_drafts(torch.zeros(1, 0, dtype=torch.int64).cuda(), None, wide, torch.zeros(1, 0, dtype=torch.float64).cuda(), us[:1])
    n, out = verify_drafts(tokens[:0], draft[:0], target[:0], ua[:0], us[:0])
    assert n.shape == (0,) and out.shape == (0, 3)
