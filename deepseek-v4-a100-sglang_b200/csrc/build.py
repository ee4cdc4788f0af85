"""Build the C-ABI shared library libdsv4_b200.so for sm_100a, in-tree.

    python build.py            # -> ../dsv4_b200/libdsv4_b200.so
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
PKG = HERE.parent / "dsv4_b200"
INCLUDE = HERE.parent.parent / "include"
LIB = PKG / "libdsv4_b200.so"
OBJ = HERE / "_build"
COMMON = [HERE / "common.cuh", HERE / "host_common.h", INCLUDE / "dsv4_b200.h"]
# translation unit -> the files it is built from
SOURCES = {
    HERE / "dsv4_b200.cu": [HERE / "gemm_tc.cuh", HERE / "small_kernels.cuh", *COMMON],
    HERE / "feed_forward.cu": [HERE / "gemm_f16.cuh", HERE / "gemm_f16_stream.cuh", HERE / "gemm_f16_rows.cuh",
                                 HERE / "feed_forward_kernels.cuh", *COMMON],
}
DEPS = [*SOURCES, *(d for deps in SOURCES.values() for d in deps)]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-v",
]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    return cand if Path(cand).exists() else "nvcc"


def up_to_date() -> bool:
    if not LIB.exists():
        return False
    t = LIB.stat().st_mtime
    return all(d.stat().st_mtime <= t for d in DEPS)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and up_to_date():
        return LIB
    PKG.mkdir(parents=True, exist_ok=True)
    OBJ.mkdir(exist_ok=True)
    jobs, objects = [], []
    for src, deps in SOURCES.items():
        obj = OBJ / (src.stem + ".o")
        objects.append(obj)
        if not force and obj.exists() and obj.with_suffix(".log").exists() and all(
                d.stat().st_mtime <= obj.stat().st_mtime for d in (src, *deps)):
            continue
        cmd = [nvcc(), *NVCC_FLAGS, "-I", str(INCLUDE), "-I", str(HERE), "-c", str(src), "-o",
               str(obj) + ".tmp"]
        jobs.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                           text=True)))
    for obj, job in jobs:
        text, _ = job.communicate()
        if job.returncode != 0:
            sys.stderr.write(text)
            raise RuntimeError(f"nvcc failed building {obj.stem}.cu")
        obj.with_suffix(".log").write_text(text)
        os.replace(str(obj) + ".tmp", obj)
    report = "".join(obj.with_suffix(".log").read_text() for obj in objects)
    if verbose:
        (HERE.parent / "ptxas_report.txt").write_text(report)
    tmp = LIB.with_suffix(".so.tmp")
    res = subprocess.run([nvcc(), "-shared", *map(str, objects), "-o", str(tmp)],
                         capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed linking libdsv4_b200.so")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
