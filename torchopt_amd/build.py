"""Compile the three in-tree binaries:

  libtoa_adam.so              the HIP kernels behind the C ABI (hipcc, gfx950 only)
  libtoa_muon.so              the same for the operators on matrix-shaped parameters
  _C.<python-abi>.so          the PyTorch extension module in front of them (g++, host only)

    python torchopt_amd/build.py

(run as a script, or load this file by path: importing the package itself needs the binaries
this file produces).  hipcc cross-compiles without a GPU, so this runs anywhere ROCm and PyTorch-ROCm are installed.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
LIB_PATH = os.path.join(PKG_DIR, 'libtoa_adam.so')
SOURCES = [os.path.join(PKG_DIR, 'csrc', 'toa_adam.hip')]
HEADERS = [
    os.path.join(PKG_DIR, 'csrc', 'adam_kernels.hpp'),
    os.path.join(PKG_DIR, 'csrc', 'plan_cache.hpp'),
    os.path.join(REPO_DIR, 'include', 'toa_adam.h'),
]
MUON_LIB_PATH = os.path.join(PKG_DIR, 'libtoa_muon.so')
MUON_SOURCES = [os.path.join(PKG_DIR, 'csrc', 'toa_muon.hip')]
MUON_HEADERS = [
    os.path.join(PKG_DIR, 'csrc', 'muon_kernels.hpp'),
    os.path.join(REPO_DIR, 'include', 'toa_muon.h'),
    os.path.join(REPO_DIR, 'include', 'toa_adam.h'),
]

# -ffp-contract=off: results are pinned to a CPU build without FMA contraction;
#   every product and sum must round on its own.
# -packed-fp32-ops off: scalar fp32 VALU code only.
# No fast-math, no denormal flushing, correctly rounded divide/sqrt (defaults).
HIPCC_FLAGS = [
    '-O3',
    '-std=c++17',
    '--offload-arch=gfx950',
    '-fPIC',
    '-shared',
    '-ffp-contract=off',
    '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
    '-fvisibility=hidden',
    '-Wall',
]


def hipcc() -> str:
    exe = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'
    if not os.path.exists(exe):
        raise RuntimeError('hipcc not found: ROCm is required to build libtoa_adam.so')
    return exe


def is_stale(lib: str = LIB_PATH, sources: list[str] = SOURCES + HEADERS) -> bool:
    if not os.path.exists(lib):
        return True
    built = os.path.getmtime(lib)
    return any(os.path.getmtime(p) > built for p in sources)


def build_library(force: bool = True, verbose: bool = False) -> str:
    """Run hipcc; returns the path of the built library."""
    if not force and not is_stale():
        return LIB_PATH
    return _hipcc(SOURCES, LIB_PATH, verbose)


def build_muon_library(force: bool = True, verbose: bool = False) -> str:
    """The same for libtoa_muon.so."""
    if not force and not is_stale(MUON_LIB_PATH, MUON_SOURCES + MUON_HEADERS):
        return MUON_LIB_PATH
    return _hipcc(MUON_SOURCES, MUON_LIB_PATH, verbose)


def _hipcc(sources: list[str], lib: str, verbose: bool) -> str:
    cmd = [hipcc(), *HIPCC_FLAGS, '-I', os.path.join(REPO_DIR, 'include'),
           '-I', os.path.join(PKG_DIR, 'csrc'), *sources, '-o', lib + '.tmp']
    if verbose:
        print(' '.join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass does not know the device-only target feature; that warning is harmless
    noise = "is not a recognized feature for this target"
    err = '\n'.join(line for line in proc.stderr.splitlines() if noise not in line)
    if proc.returncode != 0:
        raise RuntimeError(f'hipcc failed ({proc.returncode}):\n{err}')
    if verbose and err.strip():
        print(err, file=sys.stderr)
    os.replace(lib + '.tmp', lib)
    return lib


BINDING_SRCS = [os.path.join(PKG_DIR, 'csrc', f) for f in ('binding.cpp', 'binding_muon.cpp')]
BINDING_PATH = os.path.join(PKG_DIR, '_C' + sysconfig.get_config_var('EXT_SUFFIX'))


def build_binding(verbose: bool = False) -> str:
    """Compile torchopt_amd/_C*.so: pybind11 + ATen on the host side, linked against the
    libraries (found next to it at run time through an $ORIGIN rpath)."""
    import torch
    from torch.utils import cpp_extension

    if not os.path.exists(LIB_PATH):
        build_library()
    if not os.path.exists(MUON_LIB_PATH):
        build_muon_library()
    rocm = os.environ.get('ROCM_PATH', '/opt/rocm')
    torch_lib = cpp_extension.library_paths()[0]
    includes = [os.path.join(REPO_DIR, 'include'), *cpp_extension.include_paths(),
                sysconfig.get_paths()['include'], os.path.join(rocm, 'include')]
    flags = ['-O2', '-std=c++17', '-fPIC', '-fvisibility=hidden', '-Wall', '-Wno-unused-function',
             '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1', '-DTORCH_EXTENSION_NAME=_C',
             f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
             *[f'-I{p}' for p in includes]]
    cxx = os.environ.get('CXX', 'g++')
    objects = [BINDING_PATH + f'.{k}.o' for k in range(len(BINDING_SRCS))]
    try:
        # one translation unit for each submodule, compiled side by side
        _run_all([[cxx, *flags, '-c', src, '-o', obj] for src, obj in zip(BINDING_SRCS, objects)],
                 verbose)
        _run_all([[cxx, '-shared', *objects, '-o', BINDING_PATH + '.tmp',
                   f'-L{torch_lib}', f'-L{PKG_DIR}', f'-L{os.path.join(rocm, "lib")}',
                   '-ltorch_python', '-ltorch', '-ltorch_cpu', '-lc10', '-lc10_hip', '-ltorch_hip',
                   '-l:libtoa_adam.so', '-l:libtoa_muon.so', '-lamdhip64',
                   '-Wl,-rpath,$ORIGIN', f'-Wl,-rpath,{torch_lib}',
                   f'-Wl,-rpath,{os.path.join(rocm, "lib")}']], verbose)
    finally:
        for obj in objects:
            if os.path.exists(obj):
                os.remove(obj)
    os.replace(BINDING_PATH + '.tmp', BINDING_PATH)
    return BINDING_PATH


def _run_all(cmds: list[list[str]], verbose: bool) -> None:
    """Run commands side by side; all have to succeed."""
    procs = []
    for cmd in cmds:
        if verbose:
            print(' '.join(cmd), flush=True)
        procs.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE,
                                      text=True))
    for cmd, proc in zip(cmds, procs):
        err = proc.communicate()[1]
        if proc.returncode != 0:
            for other in procs:
                other.kill()
            raise RuntimeError(f'{cmd[0]} failed ({proc.returncode}):\n{err[-4000:]}')
        if verbose and err.strip():
            print(err, file=sys.stderr)


def build_all(verbose: bool = False) -> list[str]:
    return [build_library(force=True, verbose=verbose),
            build_muon_library(force=True, verbose=verbose), build_binding(verbose=verbose)]


if __name__ == '__main__':
    for path in build_all(verbose=True):
        print(path)
