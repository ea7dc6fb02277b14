"""Ahead-of-time build of the CUDA library (sm_100a only) and of the CPython extension in front of it.  `python aiter_b200/build.py` (run as a script: importing the package needs the library it produces)."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc")
LIB_PATH = os.path.join(CSRC, "libaiter_b200.so")
SOURCES = ["abi.cu", "abi_block.cu", "launch.cu", "noalloc.cu"]
HOST_PATH = os.path.join(CSRC, "_aiter_b200_host.so")
HOST_SOURCE = "host.cpp"
PUBLIC_HEADER = os.path.join("..", "..", "include", "aiter_b200.h")
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-shared", "--threads", "0",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found: the CUDA library cannot be built")
    return exe


def _host_command() -> list[str]:
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    # (no run path: torch's libraries are in the process before the extension is)
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(f"-I{p}" for p in (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"])),
            HOST_SOURCE, "-o", HOST_PATH, f"-L{os.path.join(root, 'lib')}", "-lc10", "-ltorch_cpu", "-ltorch_python"]


def _older(built: str, deps: list[str]) -> bool:
    if not os.path.exists(built):
        return True
    deps = [os.path.join(CSRC, d) for d in deps + [PUBLIC_HEADER]]
    return any(os.path.getmtime(d) > os.path.getmtime(built) for d in deps if os.path.exists(d))


def is_stale() -> bool:
    return _older(LIB_PATH, [f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".h"))]) or _older(HOST_PATH, [HOST_SOURCE])


def build_library(force: bool = False, verbose: bool = False) -> str:
    if not force and not is_stale():
        return LIB_PATH
    commands = [[_nvcc(), *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-o", LIB_PATH, *SOURCES], _host_command()]
    jobs = [subprocess.Popen(c, cwd=CSRC, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True) for c in commands]
    outputs = [j.communicate() for j in jobs]
    for command, job, (out, err) in zip(commands, jobs, outputs):
        if job.returncode != 0:
            raise RuntimeError(f"{os.path.basename(command[0])} failed:\n" + out + err)
    if verbose:
        sys.stderr.write(outputs[0][1])
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
