"""Builds libmica_w8a8.so in-tree for sm_100a (nvcc cross-compiles without a GPU), and _calls.so, the
compiled Python calls of its cache and log-probability entry points.

    python -m mica_b200.build          # or mica_b200.build.build()

The library is one translation unit (csrc/mica_w8a8.cu) linked against the static CUDA
runtime, so it does not depend on which libcudart torch happens to load. _calls.so
(csrc/calls.cpp, the host compiler) is built against the installed torch.
"""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
SRC = HERE / 'csrc' / 'mica_w8a8.cu'
OUT = HERE / 'libmica_w8a8.so'
CALLS_SRC = HERE / 'csrc' / 'calls.cpp'
CALLS = HERE / '_calls.so'
ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']
FLAGS = ['-O3', '-lineinfo', '-std=c++17', '-shared', '-Xcompiler', '-fPIC,-O2', '--expt-relaxed-constexpr']


def nvcc() -> str:
    for cand in (os.environ.get('NVCC'), shutil.which('nvcc'), '/usr/local/cuda/bin/nvcc'):
        if cand and Path(cand).exists():
            return cand
    raise FileNotFoundError('nvcc not found')


def cxx() -> str:
    """The system's g++, whose C++ runtime torch is linked with (a toolchain that links its own statically
    cannot throw through torch's libraries, so $CXX is not asked)."""
    for cand in ('/usr/bin/g++', shutil.which('g++')):
        if cand and Path(cand).exists():
            return cand
    raise FileNotFoundError('g++ not found')


def sources():
    return sorted((HERE / 'csrc').glob('*.cu*')) + sorted((HERE.parent / 'include').glob('*.h'))


def up_to_date() -> bool:
    if not OUT.is_file():
        return False
    t = OUT.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in sources())


def build_calls(force: bool = False) -> Path:
    """_calls.so against the installed torch; rebuilt when its sources or torch are newer."""
    import torch
    root = Path(torch.__file__).resolve().parent
    deps = [CALLS_SRC, *(HERE.parent / 'include').glob('*.h'), root / 'version.py']
    if not force and CALLS.is_file() and all(p.stat().st_mtime <= CALLS.stat().st_mtime for p in deps if p.is_file()):
        return CALLS
    cuda = Path(nvcc()).resolve().parents[1] / 'include'
    inc = [root / 'include', root / 'include' / 'torch' / 'csrc' / 'api' / 'include', sysconfig.get_paths()['include'], cuda]
    tmp = CALLS.with_suffix('.so.tmp')
    cmd = [cxx(), '-O2', '-std=c++17', '-fPIC', '-shared', '-DTORCH_EXTENSION_NAME=_calls',
           f'-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}', '-o', str(tmp), str(CALLS_SRC),
           *(f'-isystem{p}' for p in inc), f'-L{root / "lib"}', f'-Wl,-rpath,{root / "lib"}', '-lc10', '-lc10_cuda',
           '-ltorch_cpu', '-ltorch_python']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f'{cmd[0]} failed ({r.returncode}):\n{r.stdout}\n{r.stderr}')
    os.replace(tmp, CALLS)
    return CALLS


def build(force: bool = False, verbose: bool = False) -> Path:
    """The library, then, where torch is installed, the calls: callers of the C ABI need nvcc alone."""
    out = build_library(force, verbose)
    if importlib.util.find_spec('torch') is not None:
        build_calls(force)
    return out


def build_library(force: bool = False, verbose: bool = False) -> Path:
    if not force and up_to_date():
        return OUT
    tmp = OUT.with_suffix('.so.tmp')
    cmd = [nvcc(), *ARCH, *FLAGS, '-o', str(tmp), str(SRC)]
    if verbose:
        cmd.insert(1, '-Xptxas=-v')
        print(' '.join(cmd), file=sys.stderr)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f'nvcc failed ({r.returncode}):\n{r.stdout}\n{r.stderr}')
    if verbose:
        print(r.stderr, file=sys.stderr)
    os.replace(tmp, OUT)
    return OUT


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose='-v' in sys.argv))
