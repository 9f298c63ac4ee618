"""Builds the HIP engine in-tree: muzero_amd/libmuzero_amd.so (gfx950 only), and the host-side binding of the tensor operators
to torch, muzero_amd/_torch_calls.so."""
from __future__ import annotations

import os
import subprocess
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
LIB = os.path.join(HERE, 'libmuzero_amd.so')
OBJ_DIR = os.path.join(HERE, 'build')
TORCH_LIB = os.path.join(HERE, '_torch_calls.so')
TORCH_SOURCE = os.path.join(CSRC, 'torch_calls.cpp')
# translation units: the C ABI with the tree / fused-network kernels, the matrix-core kernels, and the tensor operators
SOURCES = ['engine.hip', 'mfma_kernels.hip', 'chain_kernels.hip', 'cached_kernels_a.hip', 'cached_kernels_b.hip',
           'cached_kernels_c.hip', 'policy_kernels.hip']
HEADERS = sorted(f for f in os.listdir(CSRC) if f.endswith('.h')) + [os.path.join('..', '..', 'include', 'muzero_amd.h')]
# -ffp-contract=off: the tree arithmetic must round exactly like the reference's NumPy expressions.
# No packed float32 instructions (v_pk_add / mul / fma_f32): some of their forms have returned wrong values now and then.
FLAGS = ['--offload-arch=gfx950', '-ffp-contract=off', '-fPIC', '-std=c++17',
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
# Optimisation level per translation unit, as measured (same box, both builds): the whole-search kernels of the matrix-core
# units are larger than the 64 KB instruction cache, and optimising for size makes them 0.7 - 0.9 % faster (TicTacToe
# 16384 x 100: 7.15 -> 7.10 ms, Atari-shaped 1024 x 200: 7.84 -> 7.78 ms); the register-resident tree kernels of
# engine.hip lose 6 % that way (CartPole 256 x 50) and stay at -O3.
# The cached-decision search kernels gain another 0.5 % from the compiler's iterative scheduler for instruction-level
# parallelism (16384 x 100: 6.768 -> 6.730 ms; "max-ilp" 6.737, "max-memory-clause" 6.816); the level-by-level kernels of
# mfma_kernels.hip lose 1.6 - 2.7 % under each of the three and keep the default scheduler.
_CACHED = '-Os -mllvm --amdgpu-sched-strategy=iterative-ilp'
OPT = {'engine.hip': '-O3', 'chain_kernels.hip': '-O3', 'cached_kernels_a.hip': _CACHED, 'cached_kernels_b.hip': _CACHED,
       'cached_kernels_c.hip': _CACHED, 'policy_kernels.hip': '-O3'}
OPT_DEFAULT = '-Os'


_POLICY = {'element_types.h', 'recurrence.h', 'distill.h', 'verify.h'}   # of the tensor operators (policy_kernels.hip)


def source_fingerprint() -> str:
    """sha256 (16 hex digits) over the compiler flags and the sources of the search engine's kernels - every .hip and .h
    under csrc/ but the tensor operators', and the public header - in name order.  Measurements that belong to one state of the kernels (HBM traffic from the counter passes) carry it, so
    that a reader can tell whether they still describe the code at hand."""
    import hashlib
    h = hashlib.sha256()
    apart = _POLICY | {'api.h', 'policy_kernels.hip'}
    opt = sorted((k, v) for k, v in OPT.items() if k not in apart)
    h.update(repr((FLAGS, opt, OPT_DEFAULT)).encode())   # the same sources built differently are other kernels
    for f in sorted(set(SOURCES + HEADERS) - apart):
        h.update(os.path.basename(f).encode())
        with open(os.path.join(CSRC, f), 'rb') as fh:
            h.update(fh.read())
    return h.hexdigest()[:16]


# headers a translation unit does NOT include (everything else counts as a dependency)
_TREE_ONLY = {'search_net.h', 'search_reg.h', 'env_step.h', 'targets.h', 'api.h'} | _POLICY
NOT_INCLUDED = {'engine.hip': {'net_mfma.h', 'search_cached.h', 'search_chain.h', 'cached_launch.h'} | _POLICY,
                'policy_kernels.hip': {os.path.basename(h) for h in HEADERS} - _POLICY - {'api.h', 'muzero_amd.h'},
                'mfma_kernels.hip': _TREE_ONLY | {'search_chain.h', 'cached_launch.h'},
                'chain_kernels.hip': _TREE_ONLY | {'search_cached.h', 'cached_launch.h'},
                'cached_kernels_a.hip': _TREE_ONLY | {'search_chain.h'},
                'cached_kernels_b.hip': _TREE_ONLY | {'search_chain.h'},
                'cached_kernels_c.hip': _TREE_ONLY | {'search_chain.h'}}


def _object(src: str, defines=()) -> str:
    tag = '_'.join(defines).replace('=', '')
    return os.path.join(OBJ_DIR, src.replace('.hip', f'{"_" + tag if tag else ""}.o'))


def _command(src: str, defines=()) -> list:
    return [os.environ.get('HIPCC', '/opt/rocm/bin/hipcc'), *FLAGS, *OPT.get(src, OPT_DEFAULT).split(), *[f'-D{x}' for x in defines], '-c',
            os.path.join(CSRC, src), '-o', _object(src, defines)]


def _recipe(target: str) -> str:
    """Where the text of the command that built `target` is kept: one built by another command is as stale as one built from
    other sources."""
    return os.path.join(OBJ_DIR, os.path.basename(target) + '.command')


def _newer_or_other(target: str, deps, command) -> bool:
    try:
        t = os.path.getmtime(target)
        with open(_recipe(target)) as fh:
            return fh.read() != repr(command) or any(os.path.getmtime(f) > t for f in deps)
    except FileNotFoundError:
        return True


def _run(target: str, command) -> None:
    os.makedirs(OBJ_DIR, exist_ok=True)
    if os.path.exists(_recipe(target)):
        os.remove(_recipe(target))
    subprocess.check_call(command)
    with open(_recipe(target), 'w') as fh:
        fh.write(repr(command))


def _stale(src: str, defines=()) -> bool:
    deps = [src] + [h for h in HEADERS if os.path.basename(h) not in NOT_INCLUDED.get(src, set())]
    return _newer_or_other(_object(src, defines), [os.path.join(CSRC, f) for f in deps], _command(src, defines))


def build_torch_calls(force: bool = False) -> str:
    """Host code only (the host compiler, torch's headers and libraries; no GPU headers)."""
    import torch
    root = os.path.dirname(torch.__file__)
    include = [os.path.join(root, 'include'), os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include'),
               sysconfig.get_paths()['include']]
    libs = os.path.join(root, 'lib')
    # the version stands in the command: a binding built against another torch is built again (and refused where it is loaded)
    command = [os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-fPIC', '-shared', '-DTORCH_EXTENSION_NAME=_torch_calls',
               '-DTORCH_API_INCLUDE_EXTENSION_H', f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
               f'-DBUILT_FOR_TORCH="{torch.__version__}"', *[f'-I{i}' for i in include], TORCH_SOURCE, '-o', TORCH_LIB, f'-L{libs}',
               f'-Wl,-rpath,{libs}', '-lc10', '-ltorch_cpu', '-ltorch_python']
    if force or _newer_or_other(TORCH_LIB, [TORCH_SOURCE, os.path.join(HERE, '..', 'include', 'muzero_amd.h')], command):
        _run(TORCH_LIB, command)
    return TORCH_LIB


def build(force: bool = False, defines=(), lib: str = LIB) -> str:
    """Compiles the translation units whose sources or command changed (all of them with `force`), in parallel, and links the shared
    library.  `defines`: extra -D flags (the diagnostic build with phase stamps uses MZ_STAMPS and another `lib`)."""
    with ThreadPoolExecutor(1) as beside:
        binding = beside.submit(build_torch_calls, force) if lib == LIB else None
        _build_library(force, defines, lib)
        if binding is not None:
            binding.result()
    return lib


def _build_library(force, defines, lib) -> None:
    todo = [s for s in SOURCES if force or _stale(s, defines)]
    if todo:
        with ThreadPoolExecutor(len(todo)) as pool:
            list(pool.map(lambda s: _run(_object(s, defines), _command(s, defines)), todo))
    objs = [_object(s, defines) for s in SOURCES]
    link = [os.environ.get('HIPCC', '/opt/rocm/bin/hipcc'), '--offload-arch=gfx950', '-shared', '-fPIC', *objs, '-o', lib]
    if todo or _newer_or_other(lib, objs, link):
        _run(lib, link)


if __name__ == '__main__':
    import sys
    force = '--changed' not in sys.argv
    if '--stamps' in sys.argv:
        print(build(force=force, defines=('MZ_STAMPS',), lib=os.path.join(HERE, 'libmuzero_amd_stamps.so')))
    else:
        print(build(force=force))
