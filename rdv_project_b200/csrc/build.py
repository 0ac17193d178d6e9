"""Builds the CUDA extension in-tree: rdv_project_b200/_lib/librdvb.so.

    python -m rdv_project_b200.csrc.build [--verbose]

nvcc cross-compiles for sm_100a (no GPU needed). The library links the CUDA
runtime statically so it has no run-time dependency beyond the driver.
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)
LIB_DIR = os.path.join(PKG, "_lib")
LIB_PATH = os.path.join(LIB_DIR, "librdvb.so")
OBJ_DIR = os.path.join(LIB_DIR, "obj")
# source -> the headers it includes (beside include/rdvb.h)
SOURCES = {
    "rdvb.cu": ["host.h", "ptx.cuh", "rng.cuh", "mlp_tc.cuh", "mlp_simt.cuh", "winograd.cuh", "winograd_f43.cuh",
                "raymarch.cuh", "transmittance.cuh", "resample.cuh", "conv_tc.cuh", "sampler.cuh", "pbvr.cuh",
                "exchange.cuh"],
    "norm.cu": ["host.h", "types.cuh", "ptx.cuh", "norm.cuh"],
    "dropout.cu": ["host.h", "types.cuh", "dropout.cuh"],
    "attention.cu": ["host.h", "types.cuh", "ptx.cuh", "attention.cuh", "attention_tc.cuh",
                     "attention_tc_grad.cuh", "attention_few.cuh"],
}


def nvcc_path() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def nvcc_flags():
    return [
        "-gencode", "arch=compute_100a,code=sm_100a",
        "-lineinfo", "-O3", "-std=c++17",
        "--expt-relaxed-constexpr",
        "-Xcompiler", "-fPIC",
        "-I", os.path.join(ROOT, "include"),
        "-I", HERE,
    ]


def _object(source: str) -> str:
    return os.path.join(OBJ_DIR, os.path.splitext(source)[0] + ".o")


def _newer(target: str, deps) -> bool:
    """Whether target is missing or older than one of deps."""
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def _deps(source: str):
    return [os.path.join(HERE, f) for f in [source, *SOURCES[source]]] + [os.path.join(ROOT, "include", "rdvb.h")]


def _stale() -> bool:
    return _newer(LIB_PATH, [d for s in SOURCES for d in _deps(s)])


def _run(cmd, verbose: bool, what: str) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"nvcc failed building {what}")
    if verbose:
        sys.stdout.write(res.stdout + res.stderr)


def build(verbose: bool = False, force: bool = False, ptxas_info: bool = False) -> str:
    """Compiles each stale source to an object (in parallel) and links the
    library; without force, sources whose object is up to date are kept."""
    if not force and not _stale():
        return LIB_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    extra = ["-Xptxas", "-v"] if ptxas_info else []
    todo = [s for s in SOURCES if force or _newer(_object(s), _deps(s))]

    def compile_one(source):
        tmp = _object(source) + ".tmp"
        _run([nvcc_path(), *nvcc_flags(), "-c", "-o", tmp, os.path.join(HERE, source), *extra],
             verbose or ptxas_info, source)
        os.replace(tmp, _object(source))

    with concurrent.futures.ThreadPoolExecutor(max_workers=max(1, len(todo))) as pool:
        list(pool.map(compile_one, todo))
    tmp = LIB_PATH + ".tmp"
    _run([nvcc_path(), *nvcc_flags(), "-shared", "-o", tmp, *[_object(s) for s in SOURCES]], verbose, "librdvb.so")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    build(verbose="--verbose" in sys.argv, force=True, ptxas_info="--ptxas" in sys.argv)
    print(LIB_PATH)
