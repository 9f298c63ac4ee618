"""CPU: what the tensor operators refuse - at the Python entry points (no CPU fallback) and at the C entry points, which check
their arguments before anything reaches a GPU."""
import ctypes

import pytest
import torch


def test_host_tensors_are_refused():
    from muzero_amd.drafts import verify_drafts
    from muzero_amd.engine import EngineError
    from muzero_amd.targets import linear_recurrence
    from muzero_amd.trainer import distillation_loss, distillation_loss_grad
    t = torch.zeros(2, 3, 4)
    with pytest.raises(EngineError, match='device tensors'):
        linear_recurrence(t, t)
    for f in (distillation_loss, distillation_loss_grad):
        with pytest.raises(EngineError, match='device tensors'):
            f(t[0], torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))
    with pytest.raises(EngineError, match='device tensors'):
        verify_drafts(torch.zeros(2, 2, dtype=torch.int64), t[:, :2], t, torch.zeros(2, 2), torch.zeros(2))


def _refused(fn, struct, text):
    from muzero_amd import engine
    assert fn(ctypes.byref(struct), None) == -1
    assert text in engine.lib().mz_last_error().decode(), engine.lib().mz_last_error()


def test_recurrence_arguments():
    from muzero_amd import engine
    L = engine.lib()
    view = engine.MzStrided(4096, 12, 4, 1)
    good = dict(type=0, B=2, D=4, reverse=0, T=3, gate=view, x=view, out=view)
    for fn in (L.mz_linear_recurrence, L.mz_linear_recurrence_backward):
        assert fn(None, None) == -1
        for change, text in ((dict(type=4), 'element type'), (dict(type=-1), 'element type'), (dict(B=0), 'sizes'), (dict(D=0), 'sizes'),
                             (dict(T=0), 'sizes'), (dict(B=1 << 20, D=1 << 20), 'sizes'), (dict(gate=engine.MzStrided()), 'null'),
                             (dict(x=engine.MzStrided()), 'null'), (dict(out=engine.MzStrided()), 'null')):
            _refused(fn, engine.MzRecurrence(**{**good, **change}), text)
    _refused(L.mz_linear_recurrence_backward, engine.MzRecurrence(**good, y=view), 'gates')
    _refused(L.mz_linear_recurrence_backward, engine.MzRecurrence(**good, out_gate=view), 'gates')


def test_distillation_arguments():
    from muzero_amd import engine
    L = engine.lib()
    good = dict(type=0, teacher_type=0, index64=1, R=2, V=9, K=3, temperature=1.0, logits=4096, logits_stride=9, index=4096,
                teacher=4096, loss=4096, grad=4096, stats=4096)
    for fn in (L.mz_distill_loss, L.mz_distill_grad, L.mz_distill_loss_grad):
        assert fn(None, None) == -1
        for change, text in ((dict(type=3), 'float32'), (dict(teacher_type=3), 'float32'), (dict(R=0), 'sizes'), (dict(V=0), 'sizes'),
                             (dict(K=0), 'sizes'), (dict(K=1025), 'sizes'), (dict(V=300000, lse=4096), 'sizes'),
                             (dict(temperature=0.0), 'temperature'), (dict(temperature=-1.0), 'temperature'),
                             (dict(temperature=float('nan')), 'temperature'), (dict(temperature=float('inf')), 'temperature'),
                             (dict(logits=None), 'null'), (dict(index=None), 'null'), (dict(teacher=None), 'null')):
            _refused(fn, engine.MzDistill(**{**good, **change}), text)
    _refused(L.mz_distill_loss, engine.MzDistill(**{**good, 'loss': None}), 'null')
    _refused(L.mz_distill_loss, engine.MzDistill(**{**good, 'stats': None}), 'null')
    _refused(L.mz_distill_grad, engine.MzDistill(**{**good, 'grad': None}), 'null')
    _refused(L.mz_distill_loss_grad, engine.MzDistill(**{**good, 'grad': None}), 'null')


def test_verification_arguments():
    from muzero_amd import engine
    L = engine.lib()
    good = dict(type=0, token64=1, B=2, K=3, V=9, tokens=4096, draft=4096, target=4096, u_accept=4096, u_sample=4096,
                accepted=4096, out=4096)
    assert L.mz_verify_drafts(None, None) == -1
    for change, text in ((dict(type=7), 'element type'), (dict(B=0), 'sizes'), (dict(K=-1), 'sizes'), (dict(V=0), 'sizes'),
                         (dict(tokens=None), 'null'), (dict(target=None), 'null'), (dict(u_accept=None), 'null'),
                         (dict(u_sample=None), 'null'), (dict(accepted=None), 'null'), (dict(out=None), 'null')):
        _refused(L.mz_verify_drafts, engine.MzVerify(**{**good, **change}), text)
