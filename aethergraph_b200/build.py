"""Builds libaethergpu.so (the CUDA kernels and the C ABI) for sm_100a, and _ops.so (the row
operators as PyTorch functions, over the C ABI), in-tree.

    python -m aethergraph_b200.build [--force] [--verbose]

nvcc cross-compiles without a GPU, so this runs on a CPU-only build machine;
the shared library lands beside this file and is what `aethergraph_b200._lib`
loads.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libaethergpu.so")
OPS = os.path.join(HERE, "_ops.so")
OPS_TORCH = os.path.join(HERE, "_ops.torch")  # the PyTorch that _ops.so was built against
SOURCES = ["api.cu", "gather.cu", "sampler.cu", "synth.cu", "loader.cu", "noalloc.cu", "hetero.cu", "hop.cu", "shard.cu",
           "hetero_loader.cu", "rewrite.cu", "hot.cu", "peer_block.cu", "reorder.cu", "workspace.cu",
           "rows.cu", "product.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC,-Wall,-Wno-unused-function", "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; libaethergpu.so cannot be built")


def _torch_version() -> str:
    """Without importing it."""
    from importlib.metadata import version

    return version("torch")


def _stale() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(OPS):
        return True
    if not os.path.exists(OPS_TORCH) or open(OPS_TORCH).read() != _torch_version():
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(OPS))
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps.append(os.path.join(HERE, "..", "include", "aethergpu.h"))
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _ops_command(host: str) -> list[str]:
    """g++ over csrc/ops_torch.cpp against the installed PyTorch; finds libaethergpu.so beside it."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    includes = [*cpp_extension.include_paths(), sysconfig.get_path("include"), os.path.join(cuda, "include")]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    return [host, "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_ops",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{i}" for i in includes),
            os.path.join(CSRC, "ops_torch.cpp"), "-o", OPS + ".tmp", f"-L{HERE}", "-l:libaethergpu.so", f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch",
            "-ltorch_python", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{libs}"]


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    nvcc = _nvcc()
    objs = []
    env = dict(os.environ)
    # The image exports CC/CXX wrappers that lack some specs; use the system g++.
    host = shutil.which("g++") or "g++"
    procs = []
    for src in SOURCES:
        obj = os.path.join(CSRC, src.rsplit(".", 1)[0] + ".o")
        cmd = [nvcc, "-ccbin", host, *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd[1:1] = ["-Xptxas", "-v"]
        procs.append((src, subprocess.Popen(cmd, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    failed = False
    for src, p in procs:
        out, _ = p.communicate()
        text = out.decode(errors="replace")
        if p.returncode != 0:
            failed = True
            sys.stderr.write(f"--- nvcc failed on {src}\n{text}\n")
        elif verbose or text.strip():
            sys.stderr.write(f"--- {src}\n{text}\n")
    if failed:
        raise RuntimeError("libaethergpu.so: compilation failed")
    link = [nvcc, "-ccbin", host, "-shared", "-gencode", "arch=compute_100a,code=sm_100a",
            "-o", LIB + ".tmp", *objs, "-lpthread"]
    r = subprocess.run(link, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    if r.returncode != 0:
        raise RuntimeError("libaethergpu.so: link failed\n" + r.stdout.decode(errors="replace"))
    os.replace(LIB + ".tmp", LIB)
    r = subprocess.run(_ops_command(host), env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    if r.returncode != 0:
        raise RuntimeError("_ops.so: compilation failed\n" + r.stdout.decode(errors="replace")[-4000:])
    os.replace(OPS + ".tmp", OPS)
    with open(OPS_TORCH, "w") as f:
        f.write(_torch_version())
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
