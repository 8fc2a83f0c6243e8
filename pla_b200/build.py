"""Ahead-of-time build of the two in-tree libraries (next to this file).

    python -m pla_b200.build [--force]

* ``libpla_b200.so``: the sm_100a kernels behind the C ABI
  (include/pla_b200.h).  nvcc cross-compiles without a GPU; this is what the
  Python package and any C/C++ host load.
* ``libpla_b200_torch.so``: the torch custom ops (``torch.ops.pla_b200.*``,
  csrc/*.cpp), plain C++ over that C ABI, compiled with g++ against the
  installed torch's headers and linked to ``libpla_b200.so`` by rpath.
"""
from __future__ import annotations

import argparse
import concurrent.futures
import glob
import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libpla_b200.so")
TORCH_OUT = os.path.join(HERE, "libpla_b200_torch.so")

NVCC_FLAGS = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
]
LINK_FLAGS = ["-shared", "-Xlinker", "-soname=libpla_b200.so"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def units() -> list[str]:
    """The CUDA translation units (compiled side by side, then linked)."""
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def sources() -> list[str]:
    return sorted(units() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h"))
                  + [os.path.join(ROOT, "include", "pla_b200.h")])


def torch_units() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cpp")))


def torch_sources() -> list[str]:
    return torch_units() + [os.path.join(ROOT, "include", "pla_b200.h")]


def up_to_date(out: str = OUT, srcs: list[str] | None = None) -> bool:
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(s) <= t for s in (sources() if srcs is None else srcs))


def _run(cmd: list[str], out: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n{r.stdout}\n{r.stderr}")
    os.replace(out + ".tmp", out)


def _compile_units(cmd: list[str], srcs: list[str], where: str, verbose: bool) -> list[str]:
    """One object per source under ``where``, the compilers running side by side."""
    objs = [os.path.join(where, os.path.basename(s) + ".o") for s in srcs]
    with concurrent.futures.ThreadPoolExecutor(len(srcs)) as pool:
        for job in [pool.submit(_run, [*cmd, "-c", s, "-o", o + ".tmp"], o, verbose) for s, o in zip(srcs, objs)]:
            job.result()
    return objs


def torch_cmds() -> tuple[list[str], list[str]]:
    """g++ compile command and link flags of libpla_b200_torch.so (torch's headers, ABI flag and libraries)."""
    import torch
    from torch.utils import cpp_extension

    cuda_home = cpp_extension.CUDA_HOME or "/usr/local/cuda"
    cmd = [shutil.which("g++") or "g++", "-std=c++17", "-O2", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    cmd += [f"-I{p}" for p in cpp_extension.include_paths()] + [f"-I{os.path.join(cuda_home, 'include')}"]
    link = [f"-L{p}" for p in cpp_extension.library_paths()] + ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch"]
    return cmd, link + [f"-L{HERE}", "-lpla_b200", "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False) -> str:
    with tempfile.TemporaryDirectory(prefix="pla_b200_build_") as where:
        if force or not up_to_date():
            objs = _compile_units([_nvcc(), *NVCC_FLAGS], units(), where, verbose)
            _run([_nvcc(), *NVCC_FLAGS, *LINK_FLAGS, "-o", OUT + ".tmp", *objs], OUT, verbose)
        if force or not up_to_date(TORCH_OUT, torch_sources() + [OUT]):
            cmd, link = torch_cmds()
            objs = _compile_units(cmd, torch_units(), where, verbose)
            _run([cmd[0], "-shared", "-o", TORCH_OUT + ".tmp", *objs, *link], TORCH_OUT, verbose)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=True))
    sys.exit(0)
