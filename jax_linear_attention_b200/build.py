"""Build ``libjla_b200.so`` in-tree with nvcc for sm_100a.

    python -m jax_linear_attention_b200.build [--force] [--verbose]

Every ``csrc/*.cu`` is compiled to an object (in parallel, only when its sources are newer than the
object) and linked into ``jax_linear_attention_b200/libjla_b200.so``; ``csrc/torch_ops.cpp`` (the torch side of the layers
whose host time matters most) becomes ``_torch_ops.so`` next to it, for the torch and the Python that run the build (without
torch, the library is all that is built). No GPU is needed to build.
"""

from __future__ import annotations

import argparse
import concurrent.futures
import glob
import importlib.util
import json
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libjla_b200.so")
TORCH_OPS = os.path.join(HERE, "_torch_ops.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas", "-v",
]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found; the CUDA kernels cannot be built")
    return path


def _newer(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src: str, obj: str, verbose: bool) -> str:
    cmd = [nvcc(), *NVCC_FLAGS, "-c", src, "-o", obj]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    log = proc.stdout + proc.stderr
    with open(obj + ".log", "w") as f:
        f.write(" ".join(cmd) + "\n" + log)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{log[-6000:]}")
    if verbose:
        print(log)
    return obj


def _torch_ops_command() -> list[str]:
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], cuda]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_torch_ops",
            "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(f for path in includes for f in ("-isystem", path)), os.path.join(CSRC, "torch_ops.cpp"), "-o", TORCH_OPS,
            *(f"-L{path}" for path in cpp_extension.library_paths()), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
            "-ltorch_python"]


def _build_torch_ops(force: bool, verbose: bool) -> None:
    """Makes ``_torch_ops.so`` where its sources are newer, or where it was made for another torch or Python or by another command
    (which its file's time does not tell: ``_torch_ops.json`` beside the objects does)."""
    import torch

    cmd = _torch_ops_command()
    command = [part.replace(HERE, "") for part in cmd]  # (the tree may be moved with what was built in it)
    made_by, note = dict(torch=torch.__version__, python=sys.version, command=command), os.path.join(OBJ, "_torch_ops.json")
    try:
        with open(note) as f:
            same = json.load(f) == made_by
    except (OSError, ValueError):
        same = False
    if same and not force and not _newer(TORCH_OPS, [cmd[cmd.index("-o") - 1], os.path.join(HERE, "..", "include", "jla_b200.h")]):
        return
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"the torch side of the layers failed to build:\n{(proc.stdout + proc.stderr)[-6000:]}")
    with open(note, "w") as f:
        json.dump(made_by, f)
    if verbose:
        print(proc.stdout + proc.stderr)


def build(force: bool = False, verbose: bool = False) -> str:
    """Makes what is out of date; returns the library's path. Where the torch side fails, the library is there all the same; a
    host without torch gets the library alone."""
    os.makedirs(OBJ, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    jobs = []
    objs = []
    for src in sources:
        obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _newer(obj, [src, *headers]):
            jobs.append((src, obj))
    stale = set(glob.glob(os.path.join(OBJ, "*.o"))) - set(objs)
    for path in stale:
        os.remove(path)
    with concurrent.futures.ThreadPoolExecutor(max_workers=8) as pool:
        glue = None
        if importlib.util.find_spec("torch") is not None:
            glue = pool.submit(_build_torch_ops, force, verbose)
        list(pool.map(lambda j: _compile(j[0], j[1], verbose), jobs))
    if jobs or stale or force or _newer(LIB, objs):
        cmd = [nvcc(), "-shared", "-o", LIB, *objs, "-lcudart"]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError("link failed:\n" + proc.stdout + proc.stderr)
    if glue is None:
        print("no torch on this host: the library alone was built, without the torch side of the layers", file=sys.stderr)
    else:
        glue.result()
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
    sys.exit(0)
