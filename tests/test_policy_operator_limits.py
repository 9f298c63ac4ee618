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


def workspace(**sizes):
    """Device bytes of a forward call: more than 0 where its record is cut into a chain, a launch of one block for every link."""
    from muzero_amd import engine
    B, T, D = sizes['B'], sizes['T'], sizes['D']
    view = engine.MzStrided(4096, T * D, D, 1)
    out = ctypes.c_int64(-1)
    a = engine.MzRecurrence(type=sizes.get('type', 0), B=B, D=D, reverse=0, T=T, gate=view, x=view, out=view)
    assert engine.lib().mz_linear_recurrence_workspace(ctypes.byref(a), 0, ctypes.byref(out)) == 0
    return out.value


def test_a_chain_has_no_more_threads_than_a_grid_takes():
    for B, D, rows, threads in ((1, 2, 256, 1024), (100, 2, 256, 1024), (1, 1, 8192, 1024), (127, 1, 8192, 1024)):
        links = ((1 << 32) - 1) // threads // B
        assert workspace(B=B, D=D, T=links * rows) > 0
        assert workspace(B=B, D=D, T=links * rows + 1) == 0
    assert workspace(B=1, D=2, T=700, type=1) > 0 and workspace(B=1, D=2, T=200) == 0
