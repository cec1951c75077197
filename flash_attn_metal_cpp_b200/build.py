"""Ahead-of-time build of the B200 attention library.

Produces, inside this package directory:
  libfa_b200.so                     C ABI (include/fa_b200.h): kernels + host dispatcher
  _flash_attn_metal.<abi>.so        pybind11 module over that C ABI
  _flash_attn_paged.<abi>.so        its paged-cache operators (pybind11 and torch;
                                    left out without a torch that has CUDA)

Every CUDA translation unit is compiled for sm_100a only
(-gencode arch=compute_100a,code=sm_100a). Objects are compiled in
parallel into _build/ and relinked only when a source is newer than the
library. Run as `python flash_attn_metal_cpp_b200/build.py [--force]`.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OBJDIR = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libfa_b200.so")
EXT = os.path.join(PKG, "_flash_attn_metal" + sysconfig.get_config_var("EXT_SUFFIX"))
EXT_PAGED = os.path.join(PKG, "_flash_attn_paged" + sysconfig.get_config_var("EXT_SUFFIX"))

CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")
NVCC = os.path.join(CUDA_HOME, "bin", "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"] + ARCH

CU_SOURCES = [
    "fa_api.cu",
    "fa_aux.cu",
    "fa_host.cu",
    "fa_fwd_simt.cu",
    "fa_fwd_sm100.cu",
    "fa_fwd_sm100_d64_causal.cu",
    "fa_fwd_sm100_d64_full.cu",
    "fa_fwd_sm100_d128_causal.cu",
    "fa_fwd_sm100_d128_full.cu",
    "fa_paged_api.cu",
    "fa_paged_cache.cu",
    "fa_paged_simt.cu",
    "fa_paged_decode_f16.cu",
    "fa_paged_decode_bf16.cu",
    "fa_paged_sm100_d64_f16.cu",
    "fa_paged_sm100_d64_bf16.cu",
    "fa_paged_sm100_d128_f16.cu",
    "fa_paged_sm100_d128_bf16.cu",
]
HEADERS = ["fa_internal.h", "fa_ptx.cuh", "fa_fwd_sm100.cuh", "fa_host.h", "fa_paged.h", "fa_paged.cuh",
           "fa_paged_decode.cuh", "fa_paged_sm100.cuh"]


def _mtime(path: str) -> float:
    return os.path.getmtime(path) if os.path.exists(path) else -1.0


def _run(cmd: list[str]) -> None:
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"build step failed: {' '.join(cmd)}\n{proc.stdout}")


def _header_mtime() -> float:
    hs = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(INCLUDE, "fa_b200.h")]
    return max(_mtime(h) for h in hs)


def _compile(src: str, force: bool) -> str:
    obj = os.path.join(OBJDIR, os.path.splitext(src)[0] + ".o")
    path = os.path.join(CSRC, src)
    if force or _mtime(obj) < max(_mtime(path), _header_mtime()):
        _run([NVCC, *NVCC_FLAGS, "-I", INCLUDE, "-c", path, "-o", obj])
    return obj


def _torch_flags() -> tuple[list[str], list[str], str] | None:
    """(compile flags, link flags, version and place) of torch's C++ interface, None without a torch that has CUDA."""
    try:
        import torch
    except ImportError:
        return None
    if torch.version.cuda is None:
        return None

    root = os.path.dirname(os.path.abspath(torch.__file__))
    inc = os.path.join(root, "include")
    cflags = ["-isystem", inc, "-isystem", os.path.join(inc, "torch", "csrc", "api", "include"),
              "-isystem", os.path.join(CUDA_HOME, "include"),
              f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    lib = os.path.join(root, "lib")
    return cflags, ["-L", lib, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python",
                    f"-Wl,-rpath,{lib}"], f"torch {torch.__version__} in {root}"


def _extension(path: str, src: str, cflags: list[str], libs: list[str], force: bool, against: str = "") -> None:
    """One pybind11 extension linked to libfa_b200.so beside it; `against` names what else it was built against."""
    import pybind11

    note = os.path.join(OBJDIR, os.path.basename(path) + ".against")
    src = os.path.join(CSRC, src)
    fresh = _mtime(path) >= max(_mtime(src), _mtime(LIB), _mtime(os.path.join(INCLUDE, "fa_b200.h")))
    if against and fresh:
        fresh = os.path.exists(note) and open(note).read() == against
    if fresh and not force:
        return
    _run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-I", pybind11.get_include(),
          "-I", sysconfig.get_paths()["include"], "-I", INCLUDE, *cflags, src, "-o", path, "-L", PKG,
          "-l:libfa_b200.so", *libs, "-Wl,-rpath,$ORIGIN"])
    if against:
        with open(note, "w") as f:
            f.write(against)


def build(force: bool = False, jobs: int | None = None) -> tuple[str, str]:
    """Compile the CUDA library and the Python extensions; return the library's and the module's path."""
    if not os.path.exists(NVCC):
        raise RuntimeError(f"nvcc not found at {NVCC}")
    os.makedirs(OBJDIR, exist_ok=True)
    jobs = jobs or max(1, min(len(CU_SOURCES), os.cpu_count() or 1))
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(lambda s: _compile(s, force), CU_SOURCES))
    if force or _mtime(LIB) < max(_mtime(o) for o in objs):
        _run([NVCC, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", LIB, *objs])

    # Two extensions over the C ABI, compiled side by side: the module itself
    # (NumPy and torch, no link to torch) and the paged-cache operators, which
    # use torch's C++ interface.
    exts = [(EXT, "bindings.cpp", [], [], force)]
    flags = _torch_flags()
    if flags is not None:
        cflags, libs, torch_is = flags
        exts.append((EXT_PAGED, "bindings_paged.cpp", cflags, libs, force, torch_is))
    else:
        print("torch with CUDA is not installed: _flash_attn_paged (the paged-cache operators) is not built", file=sys.stderr)
    with cf.ThreadPoolExecutor(max_workers=2) as ex:
        list(ex.map(lambda e: _extension(*e), exts))
    return LIB, EXT


if __name__ == "__main__":
    lib, ext = build(force="--force" in sys.argv)
    print(lib)
    print(ext)
