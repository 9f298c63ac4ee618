"""CPU: the incremental build compiles again what another command built - other flags, another torch - and nothing else.  The
compilers are stand-ins that write their output file and note their arguments."""
import os
import stat

import pytest


@pytest.fixture
def box(tmp_path, monkeypatch):
    from muzero_amd import build
    log = tmp_path / 'log'
    fake = tmp_path / 'compiler'
    fake.write_text(f'#!/bin/sh\necho "$@" >> {log}\nwhile [ $# -gt 1 ]; do [ "$1" = -o ] && : > "$2"; shift; done\n')
    fake.chmod(fake.stat().st_mode | stat.S_IXUSR)
    for name in ('HIPCC', 'CXX'):
        monkeypatch.setenv(name, str(fake))
    monkeypatch.setattr(build, 'OBJ_DIR', str(tmp_path / 'objects'))
    monkeypatch.setattr(build, 'LIB', str(tmp_path / 'lib.so'))
    monkeypatch.setattr(build, 'TORCH_LIB', str(tmp_path / 'torch.so'))

    def run(**how):
        if log.exists():
            log.unlink()
        build.build(lib=build.LIB, **how)
        return log.read_text().splitlines() if log.exists() else []
    return build, run, monkeypatch


def test_nothing_changed(box):
    build, run, _ = box
    n = len(build.SOURCES)
    assert len(run()) == n + 2          # every unit, the library, the binding
    assert run() == []
    assert len(run(force=True)) == n + 2


def test_other_flags(box):
    build, run, patch = box
    run()
    patch.setattr(build, 'FLAGS', build.FLAGS + ['-DOTHER'])
    lines = run()
    assert len(lines) == len(build.SOURCES) + 1 and sum('-DOTHER' in x for x in lines) == len(build.SOURCES)
    patch.setattr(build, 'OPT', {**build.OPT, 'policy_kernels.hip': '-O1'})
    assert len(run()) == 2 and run() == []


def test_a_failed_or_missing_object_is_built_again(box):
    build, run, _ = box
    run()
    os.remove(build._object('engine.hip'))
    assert len(run()) == 2
    os.remove(build._recipe(build._object('engine.hip')))
    assert len(run()) == 2 and run() == []


def test_another_torch(box):
    import torch
    build, run, patch = box
    run()
    patch.setattr(torch, '__version__', '0.0.1')
    lines = run()
    assert len(lines) == 1 and '0.0.1' in lines[0]


def test_a_binding_of_another_torch_is_refused(monkeypatch):
    import torch
    from muzero_amd import engine
    assert engine.torch_calls().built_for == torch.__version__
    monkeypatch.setattr(engine, '_torch_calls', None)
    monkeypatch.setattr(torch, '__version__', '0.0.1')
    with pytest.raises(engine.EngineError, match='built for torch'):
        engine.torch_calls()
