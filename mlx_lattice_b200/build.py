"""Builds ``liblattice_b200.so`` (the C-ABI library) in-tree with nvcc for sm_100a, and
``_bindings.so`` (the torch side of the differentiable operators, a caller of that ABI).

Usage: ``python -m mlx_lattice_b200.build [--force] [--verbose]``. nvcc cross-compiles
without a GPU, so this runs on any machine with the CUDA toolkit.
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

PACKAGE_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PACKAGE_DIR)
CSRC_DIR = os.path.join(PACKAGE_DIR, 'csrc')
LIBRARY_PATH = os.path.join(PACKAGE_DIR, 'liblattice_b200.so')
BINDINGS_PATH = os.path.join(PACKAGE_DIR, '_bindings.so')
# what the bindings were built against: their times say nothing about another torch or Python
BINDINGS_RECORD = os.path.join(PACKAGE_DIR, '_bindings.built-with')
BINDINGS_SOURCE = os.path.join(CSRC_DIR, 'bindings.cpp')
HEADER = os.path.join(REPO_DIR, 'include', 'lattice_b200.h')

SOURCES = (
    'relation.cu',
    'conv_direct.cu',
    'conv_tc.cu',
    'conv_tc_plan.cu',
    'conv_plan.cu',
    'order.cu',
    'voxelize.cu',
    'static_scratch.cu',
    'pool.cu',
    'feature.cu', 'align.cu',
    'row_norm.cu', 'dropout.cu', 'recurrence.cu',
    'capi.cu',
)

NVCC_FLAGS = (
    '-gencode', 'arch=compute_100a,code=sm_100a',
    '-lineinfo', '-O3', '-std=c++17', '-t', '0',
    '-Xcompiler', '-fPIC', '-shared',
)


def _nvcc() -> str:
    for candidate in (os.environ.get('NVCC'), '/usr/local/cuda/bin/nvcc', 'nvcc'):
        if candidate and (os.path.isabs(candidate) and os.path.exists(candidate)):
            return candidate
    return 'nvcc'


def _inputs() -> list[str]:
    files = [os.path.join(CSRC_DIR, name) for name in os.listdir(CSRC_DIR) if not name.endswith('.cpp')]
    return [*files, HEADER]


def _is_older(target: str, inputs: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    built = os.path.getmtime(target)
    return any(os.path.getmtime(path) > built for path in inputs)


def _bindings_environment() -> str:
    import torch

    return f'torch {torch.__version__} python {sys.version}'


def record_bindings() -> None:
    with open(BINDINGS_RECORD, 'w') as file:
        file.write(_bindings_environment())


def _bindings_are_stale() -> bool:
    if _is_older(BINDINGS_PATH, [BINDINGS_SOURCE, HEADER]) or not os.path.exists(BINDINGS_RECORD):
        return True
    with open(BINDINGS_RECORD) as file:
        return file.read() != _bindings_environment()


def is_stale() -> bool:
    return _is_older(LIBRARY_PATH, _inputs()) or _bindings_are_stale()


def _run(command: list[str], target: str, verbose: bool) -> None:
    result = subprocess.run(command, capture_output=True, text=True)
    if verbose or result.returncode != 0:
        sys.stderr.write(result.stdout)
        sys.stderr.write(result.stderr)
    if result.returncode != 0:
        raise RuntimeError(f'{os.path.basename(command[0])} failed building {os.path.basename(target)}')


def _bindings_command() -> list[str]:
    import torch

    root = os.path.dirname(torch.__file__)
    toolkit = os.path.dirname(os.path.dirname(_nvcc()))
    includes = (os.path.join(REPO_DIR, 'include'), os.path.join(root, 'include'),
                os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include'),
                os.path.join(toolkit, 'include') if toolkit else '/usr/local/cuda/include',
                sysconfig.get_paths()['include'])
    return [
        # the compiler nvcc uses: the extension shares its C++ runtime with torch and the library
        'g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-Wno-attributes',
        f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
        '-DTORCH_EXTENSION_NAME=_bindings',
        *(flag for path in includes for flag in ('-isystem' if path != includes[0] else '-I', path)),
        BINDINGS_SOURCE, '-o', BINDINGS_PATH,
        '-L', PACKAGE_DIR, '-l:liblattice_b200.so', '-Wl,-rpath,$ORIGIN',
        '-L', os.path.join(root, 'lib'), '-lc10', '-lc10_cuda', '-ltorch_cpu', '-ltorch_cuda', '-ltorch',
        '-ltorch_python',
    ]


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile every CUDA source into one shared library and the bindings beside it; returns
    the library's path."""
    if force or _is_older(LIBRARY_PATH, _inputs()):
        _run([
            _nvcc(), *NVCC_FLAGS,
            *(('-Xptxas', '-v') if verbose else ()),
            '-I', os.path.join(REPO_DIR, 'include'),
            *(os.path.join(CSRC_DIR, name) for name in SOURCES),
            '-o', LIBRARY_PATH,
        ], LIBRARY_PATH, verbose)
    if force or _bindings_are_stale():
        _run(_bindings_command(), BINDINGS_PATH, verbose)
        record_bindings()
    return LIBRARY_PATH


if __name__ == '__main__':
    print(build_library(force='--force' in sys.argv, verbose='--verbose' in sys.argv))
