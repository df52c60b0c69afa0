"""Build the native code of the package, in-tree:

* ``lib/libavey_b200.so``: the CUDA library, with nvcc for sm_100a. It exports
  only the C ABI declared in ``include/avey_b200.h``. Each source is compiled
  to an object of its own (in parallel, and only when it or a header changed)
  and the objects are linked.
* ``lib/_torch_binding.so``: the Python binding of the training and serving
  operators (host C++ against PyTorch's headers; no device code).

Usage: python -m avey_kernel_b200.csrc.build [--force] [--verbose]
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG = CSRC.parent
ROOT = PKG.parent
LIB_DIR = PKG / 'lib'
OBJ_DIR = LIB_DIR / 'build'
LIB = LIB_DIR / 'libavey_b200.so'
BINDING = LIB_DIR / '_torch_binding.so'
BINDING_SOURCE = 'torch_binding.cpp'
SOURCES = ['avey_api.cu', 'avey_bwd.cu', 'avey_optim.cu', 'avey_linear.cu']
HEADERS = ['ptx.cuh', 'common.cuh', 'norm_prepass.cuh', 'simt_kernel.cuh', 'simt2_kernel.cuh',
           'small_kernel.cuh', 'tc_kernel.cuh', 'tc_long.cuh', 'tc_tf32.cuh', 'tc_gemm.cuh', 'bwd_kernels.cuh',
           'host_api.h', 'adamw_kernels.cuh',
           'tc_linear.cuh', 'linear_steps.cuh']

NVCC_FLAGS = [
    '-gencode', 'arch=compute_100a,code=sm_100a',
    '-O3', '-lineinfo', '-std=c++17',
    '-Xcompiler', '-fPIC', '-Xcompiler', '-fvisibility=hidden',
    '--expt-relaxed-constexpr',
]


def nvcc_path() -> str:
    home = os.environ.get('CUDA_HOME', '/usr/local/cuda')
    cand = Path(home) / 'bin' / 'nvcc'
    if cand.exists():
        return str(cand)
    found = shutil.which('nvcc')
    if not found:
        raise RuntimeError('nvcc not found (set CUDA_HOME)')
    return found


PUBLIC_HEADER = ROOT / 'include' / 'avey_b200.h'


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    mtime = target.stat().st_mtime
    return any(p.stat().st_mtime > mtime for p in deps)


def _headers(source: str, seen=None) -> set:
    """The package's headers that `source` includes, directly or through others."""
    seen = set() if seen is None else seen
    for line in (CSRC / source).read_text().splitlines():
        if line.startswith('#include "'):
            name = line.split('"')[1]
            if name in HEADERS and name not in seen:
                seen.add(name)
                _headers(name, seen)
    return seen


def _deps(source: str) -> list:
    return [CSRC / source, PUBLIC_HEADER, *[CSRC / h for h in _headers(source)]]


def needs_build() -> bool:
    deps = [CSRC / s for s in SOURCES + HEADERS] + [PUBLIC_HEADER]
    return _stale(LIB, deps) or _stale(BINDING, [CSRC / BINDING_SOURCE, PUBLIC_HEADER])


def _run(cmd, verbose: bool) -> None:
    if verbose:
        print(' '.join(map(str, cmd)), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f'{Path(str(cmd[0])).name} failed with exit code {res.returncode}')
    if verbose and (res.stdout or res.stderr):
        print(res.stdout + res.stderr)


def _compile(source: str, force: bool, verbose: bool, extra) -> Path:
    obj = OBJ_DIR / (Path(source).stem + '.o')
    if force or _stale(obj, _deps(source)):
        tmp = obj.with_suffix('.o.tmp')
        _run([nvcc_path(), *NVCC_FLAGS, *extra, '-I', str(ROOT / 'include'), '-I', str(CSRC), '-c',
              str(CSRC / source), '-o', str(tmp)], verbose)
        os.replace(tmp, obj)
    return obj


def _build_binding(force: bool, verbose: bool) -> None:
    source = CSRC / BINDING_SOURCE
    if not force and not _stale(BINDING, [source, PUBLIC_HEADER]):
        return
    import torch
    inc = Path(torch.__file__).resolve().parent / 'include'
    cuda = Path(nvcc_path()).resolve().parents[1] / 'include'
    libs = Path(torch.__file__).resolve().parent / 'lib'
    tmp = BINDING.with_suffix('.so.tmp')
    _run(['g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-fvisibility=hidden',
          f'-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}',
          '-I', str(ROOT / 'include'), '-I', str(CSRC), '-isystem', str(inc), '-isystem',
          str(inc / 'torch' / 'csrc' / 'api' / 'include'), '-isystem', str(cuda), '-isystem',
          sysconfig.get_paths()['include'], str(source), '-o', str(tmp), '-L', str(libs),
          '-lc10', '-lc10_cuda', '-ltorch', '-ltorch_cpu', '-ltorch_cuda', '-ltorch_python'], verbose)
    os.replace(tmp, BINDING)


def build(force: bool = False, verbose: bool = False, extra=()) -> Path:
    """Build the library and the binding unless they are newer than every source."""
    if not force and not needs_build():
        return LIB
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    with ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as pool:
        binding = pool.submit(_build_binding, force, verbose)
        objs = list(pool.map(lambda s: _compile(s, force, verbose, extra), SOURCES))
        binding.result()
    if force or _stale(LIB, objs):
        tmp = LIB.with_suffix('.so.tmp')
        _run([nvcc_path(), *NVCC_FLAGS, '-shared', *map(str, objs), '-o', str(tmp), '-lcudart'], verbose)
        os.replace(tmp, LIB)
    return LIB


def main():
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument('--force', action='store_true')
    ap.add_argument('--verbose', action='store_true')
    ap.add_argument('--ptxas-info', action='store_true', help='print registers / spills / smem')
    args = ap.parse_args()
    extra = ['-Xptxas', '-v'] if args.ptxas_info else []
    print(build(force=args.force or args.ptxas_info, verbose=args.verbose or args.ptxas_info,
                extra=extra))


if __name__ == '__main__':
    main()
