"""Builds libloopback_b200.so (the CUDA kernels and their C ABI) in-tree with nvcc for sm_100a, and _torch_ops.so (the
C++ autograd nodes on top of it, csrc/lb_torch.cpp) with the host compiler against the installed PyTorch.

Each CUDA source of csrc/ is compiled to an object file under csrc/build/ (in parallel, and only when it or a header
changed), then the objects are linked into one shared library. The autograd nodes do not link against it: they are handed
its entry points when the package loads it.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "build")
LIB = os.path.join(HERE, "libloopback_b200.so")
TORCH_SRC = os.path.join(CSRC, "lb_torch.cpp")
TORCH_LIB = os.path.join(HERE, "_torch_ops.so")
SOURCES = ("lb_api.cu", "lb_write.cu", "lb_write_mma.cu", "lb_read_fwd.cu", "lb_read_bwd.cu", "lb_read_bwd_f32.cu", "lb_step.cu",
           "lb_noalloc.cu", "lb_peer.cu", "lb_block.cu", "lb_ffn.cu", "lb_ffn_small.cu",
           "lb_gemm_cluster.cu", "lb_gemm_kk.cu", "lb_gemm_kn.cu", "lb_gemm_mn.cu")
HEADERS = ("lb_common.cuh", "lb_kernels.h", "lb_read_bwd_impl.cuh", "lb_gemm.cuh", "lb_launch.cuh", os.path.join("..", "..", "include", "loopback_b200.h"))
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden", "-ccbin", "g++",
         "--expt-relaxed-constexpr"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA kernels of loopback_b200 cannot be built")


def sources():
    return [os.path.join(CSRC, s) for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]


def _headers_mtime() -> float:
    return max(os.path.getmtime(os.path.join(CSRC, h)) for h in HEADERS if os.path.exists(os.path.join(CSRC, h)))


def _obj_of(src: str) -> str:
    return os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")


def _stale(src: str, hdr_t: float) -> bool:
    o = _obj_of(src)
    return not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(src), hdr_t)


def _outdated(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.exists(f) and os.path.getmtime(f) > t for f in deps)


def needs_build() -> bool:
    return _outdated(LIB, sources() + [os.path.join(CSRC, h) for h in HEADERS])


def needs_torch_build() -> bool:
    return _outdated(TORCH_LIB, [TORCH_SRC, os.path.join(CSRC, HEADERS[-1])])


def build_torch_ops():
    """The autograd nodes: one C++ file against PyTorch's headers (returns the command's result)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    inc = [*cpp_extension.include_paths(), os.path.join(cpp_extension.CUDA_HOME or "/usr/local/cuda", "include"),
           sysconfig.get_paths()["include"]]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-DTORCH_EXTENSION_NAME=_torch_ops", "-DTORCH_API_INCLUDE_EXTENSION_H", *[f"-I{i}" for i in inc], TORCH_SRC, "-o", TORCH_LIB,
           f"-L{libs}", "-lc10", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-lc10_cuda", f"-Wl,-rpath,{libs}"]
    return subprocess.run(cmd, capture_output=True, text=True)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu of csrc/ for sm_100a and link them into one shared library, and the autograd nodes into another.
    Returns the kernels' path."""
    if force or needs_torch_build():
        with ThreadPoolExecutor(max_workers=1) as pool:               # beside the kernels
            job = pool.submit(build_torch_ops)
            path = _build_kernels(force, verbose)
            proc = job.result()
        if proc.returncode != 0:
            raise RuntimeError(f"g++ failed on {TORCH_SRC}:\n" + proc.stdout + proc.stderr)
        return path
    return _build_kernels(force, verbose)


def _build_kernels(force: bool, verbose: bool) -> str:
    if not force and not needs_build():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    nvcc, hdr_t = _nvcc(), _headers_mtime()
    todo = [s for s in sources() if force or _stale(s, hdr_t)]

    def compile_one(src):
        cmd = [nvcc, *ARCH, *FLAGS, "-c", src, "-o", _obj_of(src)]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        return src, subprocess.run(cmd, capture_output=True, text=True)

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(todo)))) as pool:
        for src, proc in pool.map(compile_one, todo):
            if proc.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src}:\n" + proc.stdout + proc.stderr)
            if verbose:
                print(proc.stderr)
    link = [nvcc, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-ccbin", "g++", "-cudart", "static", "-o", LIB,
            *[_obj_of(s) for s in sources()]]
    proc = subprocess.run(link, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("nvcc link failed:\n" + proc.stdout + proc.stderr)
    return LIB


if __name__ == "__main__":
    print(build(force="-f" in sys.argv or "-v" in sys.argv, verbose="-v" in sys.argv))
