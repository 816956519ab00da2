"""Builds the sm_100a backend in place: cpp_inference_train_engine_b200/libmm_cuda.so, from its
two translation units (the engine and the latent-cache operators), and _latent_torch.so, the
binding of the latter to torch tensors.

    python -m cpp_inference_train_engine_b200.build

nvcc cross-compiles for sm_100a without a GPU. The CUDA runtime is linked statically and
NCCL is opened at run time, so the library's only CUDA dependency is the driver.
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRC = [os.path.join(HERE, "csrc", f) for f in ("mm_cuda.cu", "latent.cu")]
OUT = os.path.join(HERE, "libmm_cuda.so")
TORCH_SRC = os.path.join(HERE, "csrc", "latent_torch.cpp")
TORCH_OUT = os.path.join(HERE, "_latent_torch.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def sources():
    d = os.path.join(HERE, "csrc")
    return [os.path.join(d, f) for f in os.listdir(d)] + [
        os.path.join(ROOT, "include", f) for f in os.listdir(os.path.join(ROOT, "include"))]


def up_to_date() -> bool:
    if not os.path.exists(OUT) or not os.path.exists(TORCH_OUT):
        return False
    t = min(os.path.getmtime(OUT), os.path.getmtime(TORCH_OUT))
    return all(os.path.getmtime(s) <= t for s in sources())


def torch_command():
    """g++ on the torch binding, against the installed torch's headers and libraries and the
    library beside it."""
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(NVCC), "..", "include")
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                sysconfig.get_paths()["include"], cuda]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
            *[f"-isystem{i}" for i in includes], TORCH_SRC, "-o", TORCH_OUT + ".tmp", f"-L{HERE}", "-l:libmm_cuda.so",
            f"-L{os.path.join(root, 'lib')}", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10",
            "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = True) -> str:
    if not force and up_to_date():
        return OUT
    cmd = [NVCC, *ARCH, "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
           "-Xcompiler", "-fPIC", "-shared", "-cudart", "static", "-Xptxas", "-warn-spills",
           "-t", "2", "-I", os.path.join(ROOT, "include"), *SRC, "-o", OUT + ".tmp", "-ldl", "-lpthread"]
    for out, c in ((OUT, cmd), (TORCH_OUT, torch_command())):
        if verbose:
            print(" ".join(c), flush=True)
        r = subprocess.run(c, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError(f"{c[0]} failed")
        if verbose and r.stderr.strip():
            sys.stderr.write(r.stderr)
        os.replace(out + ".tmp", out)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
