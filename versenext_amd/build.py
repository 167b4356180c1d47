"""Builds libvnx_hip.so (all HIP sources under csrc/, gfx950) and _vnx_bind.so
(csrc/bind.cpp, the Python binding of its 8-bit KV cache entries) in-tree.

Usage: python -m versenext_amd.build   (or versenext_amd.build.build_library())
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import warnings
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_NAME = "libvnx_hip.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
BIND_PATH = os.path.join(PKG_DIR, "_vnx_bind.so")
OBJ_DIR = os.path.join(PKG_DIR, "_build")

ARCH = "gfx950"

# -ffp-contract=off: every fused multiply-add in the kernels is an explicit
# fma, so the fp32 arithmetic that feeds discrete decisions is reproducible.
# -packed-fp32-ops off: no v_pk_{add,mul,fma}_f32 are generated.
HIP_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-function",
    "-Wno-unknown-pragmas",
]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: the vnx HIP library cannot be built")


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def build_bind(verbose: bool = False) -> str:
    """Compiles csrc/bind.cpp against this Python and PyTorch into BIND_PATH."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    inc = [f"-isystem{d}" for d in cpp_extension.include_paths()] + [f"-I{sysconfig.get_paths()['include']}"]
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = BIND_PATH + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DVNX_BIND_TORCH="{torch.__version__}"', *inc, os.path.join(CSRC, "bind.cpp"),
           "-o", tmp, f"-L{lib}", f"-Wl,-rpath,{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10"]
    if verbose:
        print(" ".join(cmd), flush=True)
    try:
        res = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"the binding's compiler: {e}") from e
    if res.returncode != 0:
        raise RuntimeError(f"the binding did not compile:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, BIND_PATH)
    return BIND_PATH


def build_library(verbose: bool = False, jobs: int | None = None) -> str:
    """Compiles every csrc/*.hip for gfx950 and links LIB_PATH, and the Python
    binding beside it (build_bind). Returns LIB_PATH. Without g++ or the headers
    of Python and PyTorch the library is built all the same, with a warning:
    it does not need the binding, and an older one goes."""
    hipcc = _hipcc()
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sources()
    objs = [os.path.join(OBJ_DIR, os.path.basename(s)[:-4] + ".o") for s in srcs]

    def compile_one(pair):
        src, obj = pair
        cmd = [hipcc, *HIP_FLAGS, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"hipcc failed for {src}:\n{res.stdout}\n{res.stderr}")
        return res.stderr

    jobs = jobs or min(8, os.cpu_count() or 1, len(srcs))
    with ThreadPoolExecutor(max_workers=jobs + 1) as ex:
        bind = ex.submit(build_bind, verbose)
        for warn in ex.map(compile_one, zip(srcs, objs)):
            if verbose and warn:
                print(warn, file=sys.stderr)
    tmp = LIB_PATH + ".tmp"
    cmd = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    if bind.exception() is not None:
        if os.path.exists(BIND_PATH):
            os.remove(BIND_PATH)
        warnings.warn(f"{LIB_NAME} is built, its Python binding is not: {bind.exception()}", RuntimeWarning)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(verbose="-v" in sys.argv))
