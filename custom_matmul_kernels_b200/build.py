"""Builds libfbmm.so in-tree with nvcc for sm_100a.

Run as ``python -m custom_matmul_kernels_b200.build``. The shared library lands beside
this file so that it travels with the source tree; nothing is installed elsewhere.
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_PATH = os.path.join(HERE, "libfbmm.so")
_SHARED = [os.path.join(CSRC, "fbmm_host.h"), os.path.join(CSRC, "sm100_primitives.cuh"),
           os.path.join(HERE, os.pardir, "include", "fbmm.h")]
# translation unit -> the headers it includes
UNITS = {
    os.path.join(CSRC, "fbmm_api.cu"): [os.path.join(CSRC, "fbmm_kernel.cuh"),
                                        os.path.join(CSRC, "fbmm_l1_kernel.cuh")] + _SHARED,
    os.path.join(CSRC, "fbmm_mx_api.cu"): [os.path.join(CSRC, "fbmm_mx_quant.cuh"),
                                           os.path.join(CSRC, "fbmm_mx_gemm.cuh"),
                                           os.path.join(CSRC, "fbmm_mx_pair.cuh"),
                                           os.path.join(CSRC, "fbmm_mx_rows.cuh"),
                                           os.path.join(CSRC, "fbmm_x16_gemm.cuh")] + _SHARED,
}
SOURCES = list(UNITS)
HEADERS = sorted({h for hs in UNITS.values() for h in hs})
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
]


def find_nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found; libfbmm.so cannot be built")
    return nvcc


def _older(path: str, than) -> bool:
    if not os.path.exists(path):
        return True
    built = os.path.getmtime(path)
    return any(os.path.getmtime(p) > built for p in than if os.path.exists(p))


def is_stale() -> bool:
    return _older(LIB_PATH, SOURCES + HEADERS)


def _run(cmd, verbose: bool) -> None:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if verbose:
        sys.stderr.write(proc.stderr)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + proc.stdout + proc.stderr)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the translation units that are missing or older than their sources, side by side,
    and links the library; returns its path."""
    if not force and not is_stale():
        return LIB_PATH
    nvcc = find_nvcc()
    objects = {src: os.path.splitext(src)[0] + ".o" for src in SOURCES}
    todo = [src for src in SOURCES if force or _older(objects[src], [src] + UNITS[src])]
    with concurrent.futures.ThreadPoolExecutor(max_workers=max(1, len(todo))) as pool:
        jobs = [pool.submit(_run, [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) +
                            ["-c", src, "-o", objects[src]], verbose) for src in todo]
        for job in jobs:
            job.result()
    _run([nvcc] + NVCC_FLAGS + ["-shared", "-o", LIB_PATH] + list(objects.values()), verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
