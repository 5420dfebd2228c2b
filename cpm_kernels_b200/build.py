"""Builds ``lib/libcpmk_b200.so`` from ``csrc/*.cu`` and the loadable kernel modules ``lib/gemm.fatbin`` /
``lib/gemv.fatbin`` from ``csrc/modules/*_module.cu`` with nvcc for sm_100a (cross-compiles without a GPU), and the autograd module
``lib/cpmk_torch.*.so`` from ``csrc/torch/ffn.cpp`` with the host compiler, where PyTorch is installed.

Usage: ``python -m cpm_kernels_b200.build [--force] [--verbose]``
"""
from __future__ import annotations

import glob
import importlib.metadata
import os
import subprocess
import sys

_PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_PKG, "csrc")
LIB_DIR = os.path.join(_PKG, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libcpmk_b200.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
    "--threads", "0",                      # one compilation per source file in parallel
]


def _torch_version() -> str | None:
    """Of the installed PyTorch, which need not be imported for it; None without one."""
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return None


def ext_path() -> str:
    """Path of the autograd module for the running Python and the installed PyTorch, whose C++ interface it is compiled against: another
    version of either asks for another file."""
    return os.path.join(LIB_DIR, "cpmk_torch.%s.torch-%s.so" % (sys.implementation.cache_tag, _torch_version()))


EXT_PATH = ext_path()
EXT_SOURCE = os.path.join(CSRC, "torch", "ffn.cpp")

MODULES = {"gemm": "gemm_module.cu", "gemv": "gemv_module.cu", "transpose": "transpose_module.cu"}
MODULE_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-fatbin"]


def module_path(name: str) -> str:
    """Path of the built kernel module ``name`` ("gemm", "gemv" or "transpose"): the file the reference's loader reads as
    ``cuda/<name>.fatbin`` (cpm_kernels/kernels/base.py:59-71)."""
    return os.path.join(LIB_DIR, name + ".fatbin")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _inputs() -> list[str]:
    root = os.path.dirname(_PKG)
    return sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(root, "include", "*.h")) + glob.glob(os.path.join(CSRC, "modules", "*"))


def _ext_inputs() -> list[str]:
    return [EXT_SOURCE] + glob.glob(os.path.join(os.path.dirname(_PKG), "include", "*.h"))


def _ext_is_stale() -> bool:
    if _torch_version() is None:
        return False                                     # nothing to compile it against; the library does not need it
    return not os.path.exists(EXT_PATH) or any(os.path.getmtime(p) > os.path.getmtime(EXT_PATH) for p in _ext_inputs())


def _ext_command() -> list[str]:
    """The host compiler's command for the autograd module, against the installed PyTorch's headers and libraries."""
    import sysconfig
    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), cuda, sysconfig.get_paths()["include"]]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-DTORCH_EXTENSION_NAME=cpmk_torch",
            "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI)] + ["-I" + i for i in include] + \
        ["-o", EXT_PATH, EXT_SOURCE, "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]


def is_stale() -> bool:
    if _ext_is_stale():
        return True
    if not os.path.exists(LIB_PATH) or not all(os.path.exists(module_path(n)) for n in MODULES):
        return True
    built = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(p) > built for p in _inputs())


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile the library if it is missing or older than its sources; return its path."""
    if not force and not is_stale():
        return LIB_PATH
    nvcc = os.environ.get("NVCC", "nvcc")
    os.makedirs(LIB_DIR, exist_ok=True)
    # the autograd module is compiled beside the library
    ext_cmd = _ext_command() if _ext_is_stale() or (force and _torch_version()) else None
    ext = subprocess.Popen(ext_cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) if ext_cmd else None
    try:
        _compile_cuda(nvcc, verbose)
    finally:
        ext_out = ext.communicate()[0] if ext else ""
    if ext and ext.returncode != 0:
        raise RuntimeError("%s failed:\n%s\n%s" % (ext_cmd[0], " ".join(ext_cmd), ext_out))
    # the library is written first, so a stale check against its time stamp also covers the modules
    os.utime(LIB_PATH, None)
    return LIB_PATH


def _compile_cuda(nvcc: str, verbose: bool) -> None:
    cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-o", LIB_PATH] + sources()
    proc = subprocess.run(cmd, cwd=CSRC, capture_output=True, text=True)
    if verbose:
        sys.stderr.write(proc.stderr)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n%s\n%s" % (" ".join(cmd), proc.stderr))
    for name, src in MODULES.items():
        cmd = [nvcc] + MODULE_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-o", module_path(name), os.path.join("modules", src)]
        proc = subprocess.run(cmd, cwd=CSRC, capture_output=True, text=True)
        if verbose:
            sys.stderr.write(proc.stderr)
        if proc.returncode != 0:
            raise RuntimeError("nvcc failed:\n%s\n%s" % (" ".join(cmd), proc.stderr))


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
