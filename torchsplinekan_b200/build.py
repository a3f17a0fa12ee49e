"""Builds ``lib/libkan_b200.so`` (the C-ABI library) with nvcc for sm_100a.

    python torchsplinekan_b200/build.py [--force] [--verbose]

The library has no dependency on PyTorch or on libcuda at link time; it is
loaded with ctypes.  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import concurrent.futures
import functools
import importlib.metadata
import os
import re
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB_DIR = os.path.join(PKG, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libkan_b200.so")
SOURCES = ["kan_capi.cu", "kan_simt.cu", "kan_reg.cu", "kan_dense64.cu", "kan_tc.cu", "kan_tc_edge.cu", "kan_refit.cu", "kan_collective.cu", "kan_block.cu",
           "kan_block_f32.cu", "kan_block_f64.cu", "kan_block_f16.cu", "kan_block_bf16.cu", "kan_pack.cu"]
# test-only library (operand-layout self-test); never loaded by the package
SELFTEST_SOURCE = "kan_selftest.cu"
SELFTEST_PATH = os.path.join(LIB_DIR, "libkan_b200_selftest.so")
# PyTorch operator layer (TORCH_LIBRARY + pybind + autograd node), host C++ only
EXT_SOURCES = ["kan_torch_ext.cpp", "kan_block_ext.cpp"]
EXT_HEADERS = ["kan_ext_util.h", os.path.join("..", "..", "include", "kan_b200.h")]
HEADERS = ["kan_block.h", "kan_block.cuh", "kan_block_plan.h", "kan_block_ring.cuh", "kan_device.cuh", "kan_dmma.cuh", "kan_internal.h", "kan_table.cuh", "kan_tc_ptx.cuh", "kan_tc_common.cuh", os.path.join("..", "..", "include", "kan_b200.h")]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-fvisibility=hidden"]
CXX_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_C", "-DTORCH_API_INCLUDE_EXTENSION_H"]


def _nvcc_path() -> str:
    return shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"


def _nvcc() -> str:
    cand = _nvcc_path()
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; the KAN B200 library cannot be built")
    return cand


def _cxx() -> str:
    # The system compiler, whatever $CXX says: the extension must use the same libstdc++ as the
    # interpreter's other extension modules (a toolchain that links its own copy statically breaks
    # stream formatting inside the module).
    return shutil.which("g++", path="/usr/bin:/usr/local/bin:/bin") or shutil.which("g++") or "g++"


@functools.lru_cache(maxsize=None)
def _version(compiler: str) -> str:
    return subprocess.run([compiler, "--version"], capture_output=True, text=True).stdout


def _older_than(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


# What a built file was made with besides its sources (compiler and its version, flags, torch where its headers are used) is
# kept beside the objects: files made with anything else are out of date, whatever their age.
def _stamp_path(target: str) -> str:
    return os.path.join(PKG, "build", os.path.basename(target) + ".stamp")


def _made_with(target: str):
    """The stamp of ``target``, None where there is none (built elsewhere)."""
    try:
        with open(_stamp_path(target)) as f:
            return f.read()
    except OSError:
        return None


def _make(cmd, target: str, what: str, stamp: str) -> str:
    """Runs ``cmd -o target`` and returns its messages.  ``target`` appears when it is complete, and its stamp after it."""
    os.makedirs(os.path.dirname(_stamp_path(target)), exist_ok=True)
    r = subprocess.run([*cmd, "-o", target + ".tmp"], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed for {what}:\n{r.stdout}\n{r.stderr[-6000:]}")
    os.replace(target + ".tmp", target)
    with open(_stamp_path(target) + ".tmp", "w") as f:
        f.write(stamp)
    os.replace(_stamp_path(target) + ".tmp", _stamp_path(target))
    return r.stderr


def _library_stamp() -> str:
    return "\n".join([_version(_nvcc()), *ARCH_FLAGS, *NVCC_FLAGS])


def _extension_stamp() -> str:
    return "\n".join([_version(_cxx()), importlib.metadata.version("torch"), sys.version, *CXX_FLAGS])


def _includes(src: str) -> set:
    """The repository's headers that a source includes, directly or through another one."""
    found, todo = set(), [os.path.join(CSRC, src)]
    while todo:
        at = todo.pop()
        with open(at) as f:
            names = re.findall(r'^#include "([^"]+)"', f.read(), re.M)
        for path in (os.path.normpath(os.path.join(os.path.dirname(at), n)) for n in names):
            if path not in found:
                found.add(path)
                todo.append(path)
    return found


def _stale() -> bool:
    if _older_than(LIB_PATH, [os.path.join(CSRC, s) for s in SOURCES + HEADERS]):
        return True
    made = _made_with(LIB_PATH)                     # without a compiler here its version says nothing
    return made is not None and shutil.which(_nvcc_path()) is not None and made != _library_stamp()


def ext_path() -> str:
    import sysconfig
    return os.path.join(PKG, "_C" + sysconfig.get_config_var("EXT_SUFFIX"))


def build_selftest(force: bool = False) -> str:
    """The operand-layout self-test kernel as a library of its own (loaded by the tests only)."""
    src = os.path.join(CSRC, SELFTEST_SOURCE)
    if not force and not _older_than(SELFTEST_PATH, [src, os.path.join(CSRC, "kan_tc_ptx.cuh"), os.path.join(CSRC, "kan_dmma.cuh")]):
        return SELFTEST_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    cmd = [_nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, "-shared", src, "-o", SELFTEST_PATH + ".tmp"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {SELFTEST_SOURCE}:\n{r.stdout}\n{r.stderr}")
    os.replace(SELFTEST_PATH + ".tmp", SELFTEST_PATH)
    return SELFTEST_PATH


def build_extension(force: bool = False) -> str:
    """Compiles the PyTorch operator layer (csrc/kan_torch_ext.cpp, csrc/kan_block_ext.cpp) into ``_C.<abi>.so`` beside the
    package's Python files; it links libkan_b200.so (found at run time through ``$ORIGIN/lib``)."""
    import sysconfig
    target = ext_path()
    deps = [os.path.join(CSRC, s) for s in EXT_SOURCES + EXT_HEADERS]
    stamp = _extension_stamp() if shutil.which(_cxx()) else None
    if not force and not _older_than(target, deps + [LIB_PATH]) and (stamp is None or _made_with(target) in (None, stamp)):
        return target
    import torch
    from torch.utils import cpp_extension as ce
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cudart_dir = os.path.join(os.path.dirname(torch.__file__), "..", "nvidia", "cuda_runtime", "lib")
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cudart = ["-L" + cudart_dir, "-l:libcudart.so.12", "-Wl,-rpath," + os.path.abspath(cudart_dir)] \
        if os.path.exists(os.path.join(cudart_dir, "libcudart.so.12")) else ["-L" + os.path.join(cuda_home, "lib64"), "-lcudart"]
    cxx = _cxx()
    flags = [*CXX_FLAGS, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             *["-I" + p for p in ce.include_paths()], "-I" + sysconfig.get_paths()["include"],
             "-I" + os.path.join(cuda_home, "include")]

    def compile_one(src: str) -> str:
        obj = os.path.join(PKG, "build", src.replace(".cpp", ".ext.o"))
        if force or _older_than(obj, [os.path.join(CSRC, src), *_includes(src)]) or _made_with(obj) != stamp:
            _make([cxx, *flags, "-c", os.path.join(CSRC, src)], obj, src, stamp)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=len(EXT_SOURCES)) as ex:
        objs = list(ex.map(compile_one, EXT_SOURCES))
    _make([cxx, "-shared", *objs,
           "-L" + torch_lib, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python",
           "-L" + LIB_DIR, "-lkan_b200", "-Wl,-rpath,$ORIGIN/lib", "-Wl,-rpath," + torch_lib, *cudart], target,
          "the operator layer", stamp)
    return target


def build_all(force: bool = False, verbose: bool = False) -> str:
    """Library, self-test library and operator extension, each only when out of date."""
    build_library(force, verbose)
    build_selftest(force)
    build_extension(force)
    return LIB_PATH


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compiles the CUDA sources if the library is missing or older than them."""
    if not force and not _stale():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    nvcc, stamp = _nvcc(), _library_stamp()

    def compile_one(src: str) -> str:
        obj = os.path.join(PKG, "build", src.replace(".cu", ".o"))
        if not force and not verbose and not _older_than(obj, [os.path.join(CSRC, src), *_includes(src)]) \
                and _made_with(obj) == stamp:
            return obj
        messages = _make([nvcc, *(["-Xptxas", "-v"] if verbose else []), *ARCH_FLAGS, *NVCC_FLAGS, "-c", os.path.join(CSRC, src)],
                         obj, src, stamp)
        if verbose:
            sys.stderr.write(messages)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    _make([nvcc, *ARCH_FLAGS, "-shared", *objs], LIB_PATH, "the library", stamp)
    return LIB_PATH


if __name__ == "__main__":
    print(build_all(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
