"""Build recipe of libffnerf.so (the C-ABI library in include/ffnerf.h) for B200 / sm_100a.

Compiles csrc/ffn_capi.cu (which includes the training step's kernels) and the block operators'
translation units with nvcc, side by side, and links them into ``libffnerf.so`` next to this file, then
compiles the Python module ``_ffn_ops.so`` (csrc/ffn_ops_torch.cpp: the block operators on torch
tensors), which links to it.  A unit is compiled again only when one of its sources is newer than its
object.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
SO = HERE / "libffnerf.so"
CSRC = HERE / "csrc"
BUILD = HERE / "_build"
HEADER = ROOT / "include" / "ffnerf.h"
# translation unit -> the files it includes
UNITS = {
    "ffn_capi.cu": ("ffn_step.cu", "ffn_common.cuh", "ffn_raymarch.cuh", "ffn_hashgrid.cuh", "ffn_tcgen05.cuh",
                    "ffn_step_tc.cu", "ffn_noalloc.cu", "ffn_dp.cu", "ffn_batch.cu", "ffn_probe.cu", "ffn_ops.cuh"),
    "ffn_norm.cu": ("ffn_ops.cuh",),
    "ffn_scan.cu": ("ffn_ops.cuh",),
    "ffn_experts.cu": ("ffn_ops.cuh", "ffn_tcgen05.cuh"),
}
MODULE = HERE / "_ffn_ops.so"
MODULE_SOURCE = CSRC / "ffn_ops_torch.cpp"
SOURCES = [CSRC / n for n in sorted({f for u, inc in UNITS.items() for f in (u, *inc)})] + [HEADER]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    cand = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "bin" / "nvcc"
    return str(cand) if cand.exists() else "nvcc"


def _compile(unit: str, force: bool, verbose: bool):
    """Starts the compilation of one unit; None when its object is up to date."""
    obj = BUILD / (Path(unit).stem + ".o")
    newest = max(p.stat().st_mtime for p in [CSRC / unit, HEADER, *(CSRC / f for f in UNITS[unit])])
    if obj.exists() and obj.stat().st_mtime >= newest and not force:
        return None
    cmd = [nvcc(), *NVCC_FLAGS, *(["-Xptxas=-v"] if verbose else []), f"-I{ROOT / 'include'}", "-c", str(CSRC / unit),
           "-o", str(obj.with_suffix(".o.tmp"))]
    return obj, cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def build(force: bool = False, verbose: bool = False) -> Path:
    newest = max(p.stat().st_mtime for p in SOURCES)
    if SO.exists() and SO.stat().st_mtime >= newest and not force:
        build_module(force, verbose)
        return SO
    BUILD.mkdir(exist_ok=True)
    jobs = [j for j in (_compile(u, force, verbose) for u in UNITS) if j]
    failed = []
    for obj, cmd, job in jobs:
        text, _ = job.communicate()
        if job.returncode != 0:
            failed.append(f"{' '.join(cmd)}\n{text}")
            continue
        obj.with_suffix(".o.tmp").replace(obj)
        if verbose:
            print(text)
    if failed:
        raise RuntimeError("nvcc failed:\n" + "\n".join(failed))
    tmp = SO.with_suffix(".so.tmp")
    cmd = [nvcc(), *NVCC_FLAGS, "-shared", *(str(BUILD / (Path(u).stem + ".o")) for u in UNITS), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    tmp.replace(SO)
    build_module(force, verbose)
    return SO


def build_module(force: bool = False, verbose: bool = False) -> Path:
    """The Python module of the block operators, against the installed torch."""
    import torch
    home = Path(torch.__file__).resolve().parent
    newest = max(p.stat().st_mtime for p in (MODULE_SOURCE, HEADER, home / "version.py"))
    if MODULE.exists() and MODULE.stat().st_mtime >= newest and not force:
        return MODULE
    tmp = MODULE.with_suffix(".so.tmp")
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{ROOT / 'include'}",
           f"-I{home / 'include'}", f"-I{home / 'include' / 'torch' / 'csrc' / 'api' / 'include'}", f"-I{cuda / 'include'}",
           f"-I{sysconfig.get_paths()['include']}", str(MODULE_SOURCE), "-o", str(tmp), f"-L{HERE}", "-l:libffnerf.so",
           f"-L{home / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    if verbose:
        print(res.stderr)
    tmp.replace(MODULE)
    return MODULE


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
