"""Build libpilm_cuda.so (sm_100a) from pilm_b200/csrc with nvcc, in-tree.

    python -m pilm_b200.build            # or: import pilm_b200.build; build()

and _args.so, the Python entry of the 8-bit KV cache calls (csrc/args.cpp), with g++ against
torch's headers.  The library comes first and needs nvcc alone; a host without torch, Python's
headers or a C++ compiler gets it all the same, with a warning that _args.so was left out.

Both are written next to this file so that they ship with the package and with snapshots of
the repository; they are rebuilt only when a source is newer, _args.so also when it was built
for another torch or Python.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from importlib import metadata, util
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
LIB = HERE / "libpilm_cuda.so"
ARGS = HERE / "_args.so"
ARGS_STAMP = HERE / "_build" / "args.stamp"  # what the built _args.so was built for
INCLUDE = HERE.parent / "include"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
SOURCES = ["runtime.cu", "linear.cu", "linear_tc.cu", "norm.cu", "attention.cu", "accept.cu", "mtp.cu", "f32.cu",
           "kv8_append.cu", "kv8_attention.cu"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _stale() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return any(p.stat().st_mtime > t for p in deps if p.exists())


def cxx() -> str:
    return os.environ.get("CXX") or "g++"


def args_missing() -> str:
    """What this host lacks of what _args.so is built from; empty when nothing."""
    if util.find_spec("torch") is None:
        return "torch is not installed"
    header = Path(sysconfig.get_paths()["include"]) / "Python.h"
    if not header.exists():
        return f"{header} does not exist"
    if not shutil.which(cxx().split()[0]):
        return f"no C++ compiler ({cxx()})"
    return ""


def _args_target() -> str:
    return f"torch {metadata.version('torch')} {sysconfig.get_config_var('SOABI')}"


def build_args(force: bool = False) -> Path:
    """_args.so: a Python extension module on torch's C++ API."""
    src = CSRC / "args.cpp"
    deps = [src] + list(INCLUDE.glob("*.h"))
    target = _args_target()
    if (not force and ARGS.exists() and all(p.stat().st_mtime <= ARGS.stat().st_mtime for p in deps)
            and ARGS_STAMP.exists() and ARGS_STAMP.read_text() == target):
        return ARGS
    import torch
    root = Path(torch.__file__).resolve().parent
    tmp = ARGS.with_suffix(".so.tmp")
    cmd = cxx().split() + [
        "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
        "-I", sysconfig.get_paths()["include"], "-isystem", str(root / "include"),
        "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"), str(src),
        "-L", str(root / "lib"), "-lc10", "-ltorch_cpu", "-ltorch_python", "-o", str(tmp)]
    try:
        subprocess.run(cmd, check=True)
    except subprocess.CalledProcessError as e:
        raise RuntimeError(f"{ARGS.name}, the Python entry of the 8-bit KV cache calls, did not build ({LIB.name} did): "
                           f"{' '.join(cmd)}") from e
    os.replace(tmp, ARGS)
    ARGS_STAMP.parent.mkdir(exist_ok=True)
    ARGS_STAMP.write_text(target)
    return ARGS


def build(force: bool = False, verbose: bool = False) -> Path:
    build_library(force, verbose)
    missing = args_missing()
    if missing:
        warnings.warn(f"{ARGS.name} was not built: {missing}. {LIB.name} is complete; the 8-bit KV cache calls of "
                      "pilm_b200.ckernel need both")
    else:
        build_args(force)
    return LIB


def build_library(force: bool = False, verbose: bool = False) -> Path:
    if not force and not _stale():
        return LIB
    objdir = HERE / "_build"
    objdir.mkdir(exist_ok=True)
    flags = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I", str(INCLUDE),
                    "--expt-relaxed-constexpr"]
    if verbose:
        flags += ["-Xptxas", "-v"]
    objs = []
    for src in SOURCES:
        obj = objdir / (Path(src).stem + ".o")
        cmd = [nvcc()] + flags + ["-c", str(CSRC / src), "-o", str(obj)]
        subprocess.run(cmd, check=True)
        objs.append(str(obj))
    tmp = LIB.with_suffix(".so.tmp")
    subprocess.run([nvcc()] + ARCH + ["-shared", "-o", str(tmp)] + objs, check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
