"""Build libmvdecode.so, libmvquant.so and its Python binding in-tree for sm_100a.

    python -m micro_vllm_b200.build        (from the micro-vllm_b200/ source root)

libmvdecode.so holds the decode path (include/mvdecode.h), libmvquant.so the
operators with 4-bit weights and 8-bit rows (include/mvquant.h), _mvq_binding.so
their common calls as Python functions (torch's C++ API, host code only). Both
libraries link the CUDA runtime statically and resolve the driver's tensor-map
encoder at run time, so they need only the NVIDIA driver next to them.
"""
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
CSRC_DIR = PACKAGE_DIR / 'csrc'
LIB_DIR = PACKAGE_DIR / 'lib'
LIB_PATH = LIB_DIR / 'libmvdecode.so'
QUANT_LIB_PATH = LIB_DIR / 'libmvquant.so'
BINDING_PATH = LIB_DIR / '_mvq_binding.so'
INCLUDE_DIR = PACKAGE_DIR.parents[1] / 'include'

NVCC_FLAGS = [
    '-gencode', 'arch=compute_100a,code=sm_100a',
    '-lineinfo', '-O3', '-std=c++17',
    '-Xcompiler', '-fPIC', '-Xcompiler', '-fvisibility=hidden',
    '-shared',
]


def nvcc_path() -> str:
    found = shutil.which('nvcc')
    if found:
        return found
    cuda_home = os.environ.get('CUDA_HOME', '/usr/local/cuda')
    return str(Path(cuda_home) / 'bin' / 'nvcc')


def sources():
    return sorted(CSRC_DIR.glob('*.cu')) + sorted(CSRC_DIR.glob('*.cuh'))


# Library -> the translation units it is made of and the header it implements.
LIBRARIES = {
    LIB_PATH: ([CSRC_DIR / 'mv_capi.cu'], INCLUDE_DIR / 'mvdecode.h'),
    QUANT_LIB_PATH: ([CSRC_DIR / 'mvq_capi.cu', CSRC_DIR / 'w4_linear.cu', CSRC_DIR / 'w4_wide.cu'],
                     INCLUDE_DIR / 'mvquant.h'),
    BINDING_PATH: ([CSRC_DIR / 'mvq_binding.cpp'], INCLUDE_DIR / 'mvquant.h'),
}


def _command(library: Path, tmp: Path, units, verbose: bool):
    """The compiler call that makes a library of its units."""
    if library != BINDING_PATH:
        cmd = [nvcc_path(), *NVCC_FLAGS, '-I', str(INCLUDE_DIR), '--threads', str(len(units)),
               '-o', str(tmp), *map(str, units)]
        if verbose:
            cmd.insert(1, '-Xptxas=-v')
        return cmd
    import torch
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parents[1]
    includes = [root / 'include', root / 'include/torch/csrc/api/include', cuda / 'include',
                sysconfig.get_paths()['include'], INCLUDE_DIR]
    return [os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-shared', '-fPIC', '-fvisibility=hidden',
            f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}', *(f'-I{path}' for path in includes),
            '-o', str(tmp), *map(str, units), f'-L{root / "lib"}', '-lc10', '-lc10_cuda', '-ltorch_cpu', '-ltorch_cuda',
            '-ltorch_python']


def _reached(path: Path, seen=None):
    """``path`` and the files of csrc/ that it includes."""
    seen = set() if seen is None else seen
    if path not in seen:
        seen.add(path)
        for name in re.findall(r'^#include "([^"]+)"', path.read_text(), flags=re.MULTILINE):
            if (CSRC_DIR / name).exists():
                _reached(CSRC_DIR / name, seen)
    return seen


def _library_is_stale(library: Path) -> bool:
    if not library.exists():
        return True
    units, header = LIBRARIES[library]
    built = library.stat().st_mtime
    inputs = set().union(*map(_reached, units)) | {header, Path(__file__)}
    return any(path.stat().st_mtime > built for path in inputs)


def is_stale() -> bool:
    return any(_library_is_stale(library) for library in LIBRARIES)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile each library unless it is newer than every source; return the decode library's path."""
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    running = []
    for library, (units, _) in LIBRARIES.items():
        if not force and not _library_is_stale(library):
            continue
        tmp = library.with_suffix('.so.tmp')
        cmd = _command(library, tmp, units, verbose)
        if verbose:
            print(' '.join(cmd), file=sys.stderr)
        running.append((library, tmp, cmd, subprocess.Popen(cmd)))
    codes = [process.wait() for *_, process in running]
    for (library, tmp, cmd, _), code in zip(running, codes):
        if code:
            raise subprocess.CalledProcessError(code, cmd)
        os.replace(tmp, library)
    return LIB_PATH


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose='-v' in sys.argv))
