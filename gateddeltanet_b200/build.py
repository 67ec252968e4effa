"""Build libgdn_b200.so in-tree for sm_100a.

    python -m gateddeltanet_b200.build          # or __graft_entry__.build()

nvcc compiles the CUDA kernel and the C-ABI host layer into one shared
library next to this file (gateddeltanet_b200/libgdn_b200.so), linked against
the static CUDA runtime so it does not depend on torch's copy of libcudart.
g++ compiles the torch binding of the serving operators (_ops_torch.so) where
torch is installed.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libgdn_b200.so")
SOURCES = ["gdn_decode.cu", "gdn_recurrence.cu", "gdn_batch.cu", "gdn_score.cu", "gdn_host.cu", "gdn_batch_host.cu",
           "gdn_abi_host.cpp", "gdn_delta.cu", "gdn_delta_chunk.cu",
           "gdn_logits.cu", "gdn_ops_host.cu"]
HEADERS = ["gdn_engine.h", "gdn_batch.h", "gdn_synth.h", "gdn_math.h", "gdn_ops.h", "exports.map"]
TORCH_LIB = os.path.join(HERE, "_ops_torch.so")  # the Python binding of the serving operators (ops.py)
TORCH_SOURCE = "gdn_ops_torch.cpp"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the B200 engine cannot be built")


def _stale(target: str, sources) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    deps = [os.path.join(CSRC, f) for f in sources]
    deps += [os.path.join(REPO, "include", f) for f in ("gdn_model.h", "gdn_b200.h")]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def build_torch(force: bool = False, verbose: bool = False) -> str:
    """The torch binding: host code only, against the headers of the installed
    torch. Without a torch there is nothing to bind; the library is whole without it."""
    if not force and not _stale(TORCH_LIB, [TORCH_SOURCE]):
        return TORCH_LIB
    import sysconfig
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError as e:
        print(f"no torch ({e}): the binding of gateddeltanet_b200.ops is not built", file=sys.stderr)
        return ""
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    libs = cpp_extension.library_paths()
    tmp = TORCH_LIB + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-isystem{d}" for d in cpp_extension.include_paths()], f"-isystem{os.path.join(cuda, 'include')}",
           f"-isystem{sysconfig.get_paths()['include']}", "-I", os.path.join(REPO, "include"), "-o", tmp,
           os.path.join(CSRC, TORCH_SOURCE), *[f"-L{d}" for d in libs], *[f"-Wl,-rpath,{d}" for d in libs],
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, TORCH_LIB)
    return TORCH_LIB


def build(force: bool = False, verbose: bool = False) -> str:
    build_torch(force, verbose)
    if not force and not _stale(LIB, SOURCES + HEADERS):
        return LIB
    tmp = LIB + ".tmp"
    cmd = [nvcc(), *ARCH, "-lineinfo", "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC,-O3,-ffp-contract=off",
           "-I", os.path.join(REPO, "include"), "-I", CSRC, "-o", tmp,
           *[os.path.join(CSRC, s) for s in SOURCES], "-lpthread",
           "-Xlinker", "--version-script=" + os.path.join(CSRC, "exports.map")]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
