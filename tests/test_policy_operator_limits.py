"""CPU: more of what the tensor operators' C entries refuse before anything reaches a GPU."""
import ctypes

import pytest


def refused(fn, struct, text, *more):
    from muzero_amd import engine
    assert fn(ctypes.byref(struct), *(more or (None,))) == -1
    assert text in engine.lib().mz_last_error().decode(), engine.lib().mz_last_error()


@pytest.mark.parametrize('kind', [1, 2])
def test_kept_bytes_of_a_recurrence_are_whole_words(kind):
    from muzero_amd import engine
    view = engine.MzStrided(4096, 12, 4, 1)
    for p, strides in ((4097, (16, 16, 4)), (4096, (2, 16, 4)), (4096, (16, 6, 4)), (4096, (16, 16, 1))):
        a = engine.MzRecurrence(type=kind, B=2, D=4, reverse=0, T=3, gate=view, x=view, out=view, fine=engine.MzStrided(p, *strides))
        for fn in (engine.lib().mz_linear_recurrence, engine.lib().mz_linear_recurrence_backward):
            refused(fn, a, 'multiples of 4')
