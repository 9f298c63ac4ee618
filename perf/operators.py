"""The operators around a policy that learns from the search and plays ahead of it, as cases to be timed.

Three operators: the gated linear recurrence y[t] = gate[t] * y[t-1] + x[t] over long records (returns, traces, recurrent
state) with its gradients; distillation of a policy from a teacher's top logits, loss and gradient; verification of drafted
moves against the target policy from given uniforms.  `own` False: elementary torch operations; True: the framework's calls."""
import math

import torch

own = False

TYPES = {'float64': torch.float64, 'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
SIZE = {'float64': 8, 'float32': 4, 'bfloat16': 2, 'float16': 2}


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    rec = lambda name, b, t, d, dtype, reverse, backward: dict(  # noqa: E731
        name=name, op='recurrence', b=b, t=t, d=d, dtype=dtype, reverse=reverse, backward=backward)
    dis = lambda name, r, v, k, dtype, tail, fused: dict(  # noqa: E731
        name=name, op='distill', r=r, v=v, k=k, dtype=dtype, tail=tail, fused=fused)
    ver = lambda name, b, k, v, dtype: dict(name=name, op='verify', b=b, k=k, v=v, dtype=dtype)  # noqa: E731
    return [
        # lambda returns of a self-play window: 200 moves of 8192 environments, time-major float64 as the move log holds it
        rec('rec_log', 1, 200, 8192, 'float64', True, False),
        # one step of a recurrent policy that serves 64 games
        rec('rec_step', 64, 1, 2560, 'bfloat16', False, False),
        # a batch of long records read once (evaluation, prefill)
        rec('rec_read', 8, 4096, 2048, 'bfloat16', False, False),
        # the same kind of layer in training: forward and all gradients
        rec('rec_train', 4, 8192, 4096, 'bfloat16', False, True),
        # a single very long record of few, odd channels
        rec('rec_long', 1, 50000, 1000, 'float32', False, False),
        # differentiable returns of 1000 stored games of odd length, each contiguous in time
        rec('rec_rows', 1000, 4097, 1, 'float32', True, True),
        # the unrolled policy heads of a 16384-position batch over 9 actions, four of them searched
        dis('distill_board', 98304, 9, 4, 'float32', False, False),
        # a policy over a token-sized action set, loss and gradient in one call
        dis('distill_vocab', 4096, 32000, 32, 'bfloat16', False, True),
        # an odd, very wide action set with the teacher's remaining mass kept
        dis('distill_wide', 1023, 131071, 64, 'bfloat16', True, False),
        # five moves drafted ahead in every game of a 16384-game batch
        ver('verify_board', 16384, 5, 9, 'float64'),
        # one game over a token-sized action set: latency
        ver('verify_one', 1, 4, 32000, 'float32'),
        # a serving batch over a wide, odd action set
        ver('verify_batch', 256, 7, 100003, 'float32'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('recurrence', 'recurrence', 'distill', 'verify'))
    if op == 'recurrence':
        dtype = rng.choice(('float64', 'float32', 'bfloat16', 'float16'))
        d = 1 if rng.random() < 0.25 else _log(rng, 2, 8192)
        t = 1 if rng.random() < 0.15 else _log(rng, 2, 65536)
        most = 1 << 25
        b = _log(rng, 1, max(1, min(4096, most // (t * d))))
        t = max(1, min(t, most // (b * d)))
        return dict(op=op, b=b, t=t, d=d, dtype=dtype, reverse=rng.random() < 0.5, backward=rng.random() < 0.5)
    if op == 'distill':
        v = _log(rng, 2, 140000)
        k = min(v, _log(rng, 1, 128))
        r = _log(rng, 1, min(100000, (1 << 26) // v))
        return dict(op=op, r=r, v=v, k=k, dtype=rng.choice(('float32', 'bfloat16', 'float16')), tail=rng.random() < 0.5,
                    fused=rng.random() < 0.5)
    v = _log(rng, 2, 130000)
    k = rng.randint(0, 12)
    b = _log(rng, 1, max(1, min(16384, (1 << 27) // (v * (k + 1)))))
    return dict(op=op, b=b, k=k, v=v, dtype=rng.choice(('float64', 'float32', 'bfloat16', 'float16')))


# ---------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt = TYPES[case['dtype']]
    rand = lambda *s, dtype=torch.float32: torch.rand(s, generator=g, device='cuda', dtype=dtype)  # noqa: E731
    randn = lambda *s: torch.randn(s, generator=g, device='cuda')  # noqa: E731
    if case['op'] == 'recurrence':
        b, t, d = case['b'], case['t'], case['d']
        gate = torch.sigmoid(randn(b, t, d) * 1.5 + 2.5)   # memories of a few to a few hundred steps
        gate = torch.where(rand(b, t, d) < 0.01, torch.zeros((), device='cuda'), gate).to(dt)   # ends of games
        leaf = case['backward']
        return dict(case=case, gate=gate.requires_grad_(leaf), x=randn(b, t, d).to(dt).requires_grad_(leaf),
                    state=randn(b, d).to(torch.float64 if dt == torch.float64 else torch.float32).requires_grad_(leaf),
                    grad=randn(b, t, d).to(dt) if leaf else None)
    if case['op'] == 'distill':
        r, v, k = case['r'], case['v'], case['k']
        logits = (randn(r, v) * 2.5).to(dt)
        teacher = logits.float() + randn(r, v)
        top, index = torch.topk(teacher, k, dim=1)
        tau = 2.0 if case['tail'] else 1.0
        lse = torch.logsumexp(teacher / tau, dim=1)
        del teacher
        weight = torch.where(rand(r) < 0.05, torch.zeros((), device='cuda'), 0.5 + rand(r))   # padded positions weigh nothing
        if not case['tail']:
            index = torch.where(rand(r, k) < 0.05, torch.full((), -1, device='cuda', dtype=index.dtype), index)   # absent entries
        return dict(case=case, logits=logits.requires_grad_(not case['fused']), index=index, teacher=top.to(dt), tau=tau,
                    lse=lse if case['tail'] else None, weight=weight, grad=(0.5 + rand(r)) / r)
    b, k, v = case['b'], case['k'], case['v']
    z = randn(b, k + 1, v) * 2.0
    target = torch.softmax(z, dim=2).to(dt)
    draft = torch.softmax(z[:, :k] + 0.7 * randn(b, k, v), dim=2)
    del z
    if k:
        tokens = torch.multinomial(draft.reshape(b * k, v), 1, generator=g).reshape(b, k)
    else:
        tokens = torch.zeros((b, 0), dtype=torch.int64, device='cuda')
    lengths = torch.randint(0, k + 1, (b,), generator=g, device='cuda', dtype=torch.int32)
    lengths = torch.where(rand(b) < 0.75, torch.full_like(lengths, k), lengths)   # most drafts run to their full length
    return dict(case=case, tokens=tokens, draft=draft.to(dt), target=target, u_accept=rand(b, k, dtype=torch.float64),
                u_sample=rand(b, dtype=torch.float64), lengths=lengths)


# ---------------------------------------------------------------------------------------------------- one pass
def _scan(gate, x):
    """y[t] = gate[t] * y[t-1] + x[t] along axis 1 by doubling: after a step every y[t] covers twice the elements."""
    step = 1
    while step < x.shape[1]:
        x = torch.cat([x[:, :step], x[:, step:] + gate[:, step:] * x[:, :-step]], dim=1)
        gate = torch.cat([gate[:, :step], gate[:, step:] * gate[:, :-step]], dim=1)
        step *= 2
    return x


def _recurrence(s):
    case, dt = s['case'], s['x'].dtype
    wide = torch.float64 if dt == torch.float64 else torch.float32
    turn = (lambda z: z.flip(1)) if case['reverse'] else (lambda z: z)
    gate, x, state = turn(s['gate'].detach().to(wide)), turn(s['x'].detach().to(wide)), s['state'].detach()
    first = x[:, :1] + gate[:, :1] * state[:, None]
    y = _scan(gate, torch.cat([first, x[:, 1:]], dim=1))
    out = dict(y=turn(y).to(dt), state=y[:, -1].clone())
    if case['backward']:
        dy = turn(s['grad'].to(wide))
        later = torch.cat([torch.zeros_like(gate[:, :1]), gate[:, 1:].flip(1)], dim=1)   # gate[t+1], the last one's is none
        dx = _scan(later, dy.flip(1)).flip(1)
        before = torch.cat([state[:, None], y[:, :-1]], dim=1)
        out.update(dx=turn(dx).to(dt), dgate=turn(dx * before).to(dt), dstate=gate[:, 0] * dx[:, 0])
    return out


def _distill(s):
    tau, index, dt = s['tau'], s['index'], s['logits'].dtype
    z = s['logits'].detach().float() / tau
    z = z - z.amax(dim=1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(dim=1, keepdim=True, dtype=torch.float64)   # long sums in 64 bits: what is left of the mass is a difference of them
    q = e / total.float()
    there = index >= 0
    at = index.clamp(min=0)
    t = torch.where(there, s['teacher'].double() / tau, -math.inf)
    if s['lse'] is None:
        t = t - t.amax(dim=1, keepdim=True).clamp(min=-1e300)
        p = torch.exp(t)
        mass = p.sum(dim=1, keepdim=True)
        p = p / torch.where(mass > 0, mass, 1.0)
        logp = t - torch.log(torch.where(mass > 0, mass, 1.0))
    else:
        logp = t - s['lse'].double()[:, None]
        p = torch.exp(logp)
    some = there.any(dim=1)
    logq = z.gather(1, at).double() - torch.log(total)
    taken = torch.where(p > 0, p * (logp - logq), 0.0).sum(dim=1)
    mass = p.sum(dim=1, keepdim=True).float()
    grad = q * mass
    if s['lse'] is not None:
        inside = torch.zeros_like(z, dtype=torch.bool).scatter(1, at, True)
        qrest = torch.where(inside, 0.0, e).sum(dim=1, keepdim=True, dtype=torch.float64) / total
        # without an action outside the entries there is no remaining mass to compare
        rest = torch.where(qrest > 0, (1.0 - p.sum(dim=1, keepdim=True)).clamp(min=0.0), 0.0)
        ratio = rest / torch.where(qrest > 0, qrest, 1.0)
        taken = taken + torch.where(rest > 0, rest * torch.log(ratio), 0.0)[:, 0]
        grad = q * torch.where(inside, mass + rest.float(), (mass.double() + rest - ratio).float())
    grad = grad.scatter_add(1, at, -p.float())
    weight = torch.where(some, s['weight'], 0.0)
    loss = torch.where(weight != 0, weight.double() * tau * tau * taken, 0.0).float()
    scale = weight * tau if s['case']['fused'] else weight * tau * s['grad']
    return dict(loss=loss, grad=torch.where(scale[:, None] != 0, scale[:, None] * grad, 0.0).to(dt))


def _verify(s):
    tokens, u = s['tokens'], s['u_accept']
    b, k = tokens.shape
    row = torch.arange(b, device='cuda')
    step = torch.arange(k, device='cuda')
    pt = s['target'][:, :k].gather(2, tokens[:, :, None])[:, :, 0].double()
    qt = s['draft'].gather(2, tokens[:, :, None])[:, :, 0].double()
    ok = (u * qt < pt) & (step < s['lengths'][:, None])
    n = ok.int().cumprod(dim=1).sum(dim=1)
    left = s['target'][row, n].double()
    if k:
        rejected = (n < s['lengths'])[:, None]
        less = (left - s['draft'][row, n.clamp(max=k - 1)].double()).clamp(min=0.0)
        left = torch.where(rejected & (less.amax(dim=1, keepdim=True) > 0), less, left)
    sums = left.cumsum(dim=1)
    token = (sums <= s['u_sample'][:, None] * sums[:, -1:]).sum(dim=1)
    last = torch.where(left > 0, torch.arange(left.shape[1], device='cuda'), -1).amax(dim=1)
    token = torch.minimum(token, last)
    out = torch.full((b, k + 1), -1, dtype=tokens.dtype, device='cuda')
    out[:, :k] = torch.where(step < n[:, None], tokens, -1)
    return dict(accepted=n.int(), tokens=out.scatter(1, n[:, None], token[:, None]))


def run(state):
    s, case = state, state['case']
    if case['op'] == 'recurrence':
        if not own:
            return _recurrence(s)
        from muzero_amd.targets import linear_recurrence
        y, last = linear_recurrence(s['gate'], s['x'], s['state'], reverse=case['reverse'])
        if not case['backward']:
            return dict(y=y, state=last)
        dx, dgate, dstate = torch.autograd.grad(y, (s['x'], s['gate'], s['state']), s['grad'])
        return dict(y=y, state=last, dx=dx, dgate=dgate, dstate=dstate)
    if case['op'] == 'distill':
        if not own:
            return _distill(s)
        from muzero_amd.trainer import distillation_loss, distillation_loss_grad
        if case['fused']:
            loss, grad = distillation_loss_grad(s['logits'], s['index'], s['teacher'], teacher_lse=s['lse'],
                                                temperature=s['tau'], weight=s['weight'])
            return dict(loss=loss, grad=grad)
        loss = distillation_loss(s['logits'], s['index'], s['teacher'], teacher_lse=s['lse'], temperature=s['tau'],
                                 weight=s['weight'])
        grad, = torch.autograd.grad(loss, (s['logits'],), s['grad'])
        return dict(loss=loss, grad=grad)
    if not own:
        return _verify(s)
    from muzero_amd.drafts import verify_drafts
    accepted, tokens = verify_drafts(s['tokens'], s['draft'], s['target'], s['u_accept'], s['u_sample'], lengths=s['lengths'])
    return dict(accepted=accepted, tokens=tokens)


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = SIZE[case['dtype']]
    if case['op'] == 'recurrence':
        n, rows = case['b'] * case['t'] * case['d'], case['b'] * case['d']
        state = 8 if size == 8 else 4
        # gate, x in, y out, both states; in training the incoming gradient in, two gradients out, the state's out
        return dict(bytes=n * size * (6 if case['backward'] else 3) + rows * state * (3 if case['backward'] else 2),
                    flops=n * (5 if case['backward'] else 2))
    if case['op'] == 'distill':
        n = case['r'] * case['v']
        return dict(bytes=2 * n * size + case['r'] * (case['k'] * (size + 8) + 12 + 4 * case['tail']), flops=6 * n)
    b, k, v = case['b'], case['k'], case['v']
    # one row of each policy, the drafted tokens' entries, the uniforms, the answer
    return dict(bytes=b * (2 * v * size + k * (2 * size + 16) + 8 + 4 + 4 + 8 * (k + 1)), flops=3 * b * v)


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'recurrence':
        a, x, h = s['gate'].detach().double(), s['x'].detach().double(), s['state'].detach().double()
        order = range(case['t'])[::-1] if case['reverse'] else range(case['t'])
        y, before = torch.empty_like(x), torch.empty_like(x)
        for t in order:
            before[:, t] = h
            h = torch.addcmul(x[:, t], a[:, t], h)
            y[:, t] = h
        out = dict(y=y, state=h)
        if case['backward']:
            dx, carry = s['grad'].double(), torch.zeros_like(h)
            for t in reversed(order):
                dx[:, t] += carry
                carry = a[:, t] * dx[:, t]
            out.update(dx=dx, dgate=dx * before, dstate=carry)
        return out
    if case['op'] == 'verify':
        return None   # whole numbers
    losses, grads = [], []
    rows = max(1, (1 << 25) // case['v'])
    for i in range(0, case['r'], rows):   # autograd of the definition, some rows at a time
        part = slice(i, min(i + rows, case['r']))
        z = s['logits'].detach()[part].double().requires_grad_()
        logq = torch.log_softmax(z / s['tau'], dim=1)
        p = torch.zeros_like(logq)
        there = s['index'][part] >= 0
        at = s['index'][part].clamp(min=0)
        t = torch.where(there, s['teacher'][part].double() / s['tau'], -math.inf)
        if s['lse'] is None:
            some = there.any(dim=1, keepdim=True)
            pk = torch.where(some, torch.softmax(torch.where(some, t, 0.0), dim=1), 0.0)
        else:
            pk = torch.exp(t - s['lse'][part].double()[:, None])
        p.scatter_add_(1, at, pk)
        kl = torch.special.entr(p).neg().sum(dim=1) - (p * logq).sum(dim=1)
        if s['lse'] is not None:
            inside = torch.zeros_like(p, dtype=torch.bool).scatter_(1, at, there)
            rest = (1.0 - p.sum(dim=1)).clamp(min=0.0)
            logrest = torch.logsumexp(logq.masked_fill(inside, -math.inf), dim=1)
            kl = kl + torch.where(torch.isfinite(logrest), -torch.special.entr(rest) - rest * logrest, 0.0)
        loss = s['weight'][part].double() * s['tau'] ** 2 * kl
        up = torch.ones_like(loss) if case['fused'] else s['grad'][part].double()
        grad, = torch.autograd.grad(loss, z, up)
        losses.append(loss.detach())
        grads.append(grad)
    return dict(loss=torch.cat(losses), grad=torch.cat(grads))
