"""Build libad_b200.so in-tree with nvcc for sm_100a.

``python -m ad_b200.build`` (also called by ``__graft_entry__.build()``).
The library links the CUDA runtime statically and NVRTC dynamically; the CUDA
driver is reached through ``cudaGetDriverEntryPoint`` and NCCL is dlopen'ed, so
the library loads on a machine without a GPU driver.
"""
import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
LIB = os.path.join(PKG, "libad_b200.so")
SOURCES = [os.path.join(PKG, "csrc", f) for f in (
    "runtime.cu", "noalloc.cu", "rotary.cu", "block_norm.cu", "block_norm_f32.cu", "block_norm_bf16.cu",
    "block_norm_f16.cu", "token_logprobs.cu", "orthogonalize.cu")]
HEADERS = [os.path.join(ROOT, "include", "ad_b200.h"), os.path.join(PKG, "csrc", "ops_common.cuh"),
           os.path.join(PKG, "csrc", "block_norm.cuh")]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(s) > t for s in SOURCES + HEADERS)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    tmp = LIB + f".{os.getpid()}.tmp"
    flags = ["-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
             "-Xcompiler", "-fPIC", "-I", os.path.join(ROOT, "include")]

    def run(cmd):
        if verbose:
            print(" ".join(cmd))
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + r.stdout[-3000:] + r.stderr[-6000:])

    # one object a source, side by side
    with tempfile.TemporaryDirectory() as d, ThreadPoolExecutor(os.cpu_count() or 4) as pool:
        objects = [os.path.join(d, os.path.basename(s) + ".o") for s in SOURCES]
        list(pool.map(lambda so: run([NVCC, *flags, "-c", so[0], "-o", so[1]]), zip(SOURCES, objects)))
        run([NVCC, *flags, "-shared", "-cudart", "static", *objects, "-o", tmp, "-lnvrtc", "-ldl", "-lpthread"])
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
