"""Build the sm_100a CUDA library (libbitnet_b200.so) in-tree with nvcc, and the
Python module of the paged cache's calls (_paged.so) with g++.

The library is one translation unit (csrc/capi.cu includes every kernel
header), compiled for sm_100a only and linked against the static CUDA runtime,
so the .so has no dependency beyond the driver and travels with the source tree.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)  # .../bitnet-tt_b200
CSRC = os.path.join(ROOT, "csrc")
LIB_NAME = "libbitnet_b200.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared", "-cudart", "static",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the B200 library cannot be built")


def _sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    lib_mtime = os.path.getmtime(LIB_PATH)
    header = os.path.join(os.path.dirname(ROOT), "include", "bitnet_b200.h")
    deps = _sources() + ([header] if os.path.exists(header) else [])
    return any(os.path.getmtime(s) > lib_mtime for s in deps)


EXT_PATH = os.path.join(PKG_DIR, "_paged.so")
EXT_SOURCE = os.path.join(CSRC, "paged_binding.cpp")


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """Compile csrc/paged_binding.cpp against torch's headers and libbitnet_b200.so
    (found beside it at run time) into bitnet_tt/_paged.so; return its path."""
    header = os.path.join(os.path.dirname(ROOT), "include", "bitnet_b200.h")
    deps = [p for p in (EXT_SOURCE, header) if os.path.exists(p)]
    import torch
    from torch.utils import cpp_extension

    # torch's headers are not among the sources whose times count: another torch means another build
    stamp = EXT_PATH + ".stamp"
    made_for = f"torch {torch.__version__}, python {sysconfig.get_python_version()}\n"
    if not force and os.path.exists(EXT_PATH) and all(os.path.getmtime(d) <= os.path.getmtime(EXT_PATH) for d in deps):
        if os.path.exists(stamp) and open(stamp).read() == made_for:
            return EXT_PATH
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    inc = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = EXT_PATH + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{i}" for i in inc], EXT_SOURCE,
           "-o", tmp, f"-L{lib}", f"-Wl,-rpath,{lib}", "-Wl,-rpath,$ORIGIN", "-ltorch_python", "-ltorch_cpu", "-ltorch",
           "-lc10", "-lc10_cuda", f"-L{PKG_DIR}", f"-l:{LIB_NAME}"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, EXT_PATH)
    with open(stamp, "w") as f:
        f.write(made_for)
    return EXT_PATH


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    """Compile csrc/capi.cu into bitnet_tt/libbitnet_b200.so, and the binding beside
    it; return the library's path."""
    if not force and not needs_build():
        build_binding(verbose=verbose)
        return LIB_PATH
    tmp = LIB_PATH + ".tmp"
    cmd = [_nvcc(), *NVCC_FLAGS]
    if ptxas_info:
        cmd += ["-Xptxas", "-v"]
    cmd += ["-o", tmp, os.path.join(CSRC, "capi.cu")]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    if verbose or ptxas_info:
        sys.stderr.write(proc.stdout + proc.stderr)
    os.replace(tmp, LIB_PATH)
    build_binding(force=force, verbose=verbose)
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas" in sys.argv)
