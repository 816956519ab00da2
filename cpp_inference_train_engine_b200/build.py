"""Builds the sm_100a backend in place: cpp_inference_train_engine_b200/libmm_cuda.so, from its
two translation units (the engine and the latent-cache operators), and after it _latent_torch.so,
the binding of the latter to torch tensors, where a torch with CUDA can be imported (the library
needs none).

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


def up_to_date(out: str) -> bool:
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(s) <= t for s in sources())


def torch_command():
    """g++ on the torch binding, against the installed torch's headers and libraries and the
    library beside it. ImportError where there is no torch with CUDA."""
    import sysconfig

    import torch
    if not torch.version.cuda:
        raise ImportError("the installed torch has no CUDA")
    root = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(NVCC), "..", "include")
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                sysconfig.get_paths()["include"], cuda]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
            *[f"-isystem{i}" for i in includes], TORCH_SRC, "-o", TORCH_OUT + ".tmp", f"-L{HERE}", "-l:libmm_cuda.so",
            f"-L{os.path.join(root, 'lib')}", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10",
            "-Wl,-rpath,$ORIGIN"]


def _run(command, out: str, verbose: bool) -> None:
    """A compiler that writes out + ".tmp", put in place when it succeeds."""
    if verbose:
        print(" ".join(command), flush=True)
    r = subprocess.run(command, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"{command[0]} failed")
    if verbose and r.stderr.strip():
        sys.stderr.write(r.stderr)
    os.replace(out + ".tmp", out)


def build(force: bool = False, verbose: bool = True) -> str:
    if force or not up_to_date(OUT):
        _run([NVCC, *ARCH, "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
              "-Xcompiler", "-fPIC", "-shared", "-cudart", "static", "-Xptxas", "-warn-spills",
              "-t", "2", "-I", os.path.join(ROOT, "include"), *SRC, "-o", OUT + ".tmp", "-ldl", "-lpthread"], OUT, verbose)
    if force or not up_to_date(TORCH_OUT):
        try:
            command = torch_command()
        except ImportError as e:
            sys.stderr.write(f"{os.path.basename(TORCH_OUT)} (latent.py) was not built, it needs a torch with CUDA: {e}\n")
        else:
            _run(command, TORCH_OUT, verbose)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
