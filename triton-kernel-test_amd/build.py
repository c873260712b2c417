"""Build liblrq.so (the HIP kernels + C ABI) for gfx950 with hipcc, in-tree.

Usage: python triton-kernel-test_amd/build.py [--jobs N]

Objects go to triton-kernel-test_amd/_build/, the library to
triton-kernel-test_amd/liblrq.so.  Every source is rebuilt on each call (the build
check wants a real compile); compiles run in parallel.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "liblrq.so"
ARCH = "gfx950"

# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 are generated (the host pass warns that
# it does not know the feature; that is harmless).
HIPFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-ffp-contract=off",
    # MFMA results straight into VGPRs (no v_accvgpr_read round trips in the epilogues)
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    # every masked region restores its own mask.  Where two regions end together the compiler would leave out the inner
    # restore, and spilled registers reloaded between the two ends then miss the lanes that skipped the inner region: a row
    # loop whose step was reloaded so never ended.  Costs a scalar instruction a region: times are the same within noise.
    "-mllvm", "-amdgpu-remove-redundant-endcf=0",
]

# The compressed format assumes finite inputs (NaN / Inf activations give unspecified codes, never a fault).  IEEE mode
# off: v_min/v_max of MFMA results need no canonicalising moves.
FINITE_FLAGS = ["-fno-honor-nans", "-mno-amdgpu-ieee"]

# The layer norm, dropout and MXFP4 kernels carry NaN and infinity through their row or block.  Without NaNs honoured
# every operation on one would be undefined to the compiler, so these are built with the language's own arithmetic.
CARRY_NAN = {"lrq_dropout", "lrq_mx", "lrq_mxgemm", "lrq_norm_bwd", "lrq_norm_fwd"}


def flags(src: Path) -> list[str]:
    return HIPFLAGS if src.stem in CARRY_NAN else HIPFLAGS + FINITE_FLAGS


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (ROCm is required to build liblrq.so)")


def _compile(src: Path) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [hipcc(), *flags(src), "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in (res.stderr or "").splitlines() if noise not in l)
    if res.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{err}")
    if err.strip():
        print(err, file=sys.stderr)
    return obj


def build(jobs: int | None = None, verbose: bool = True) -> Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    jobs = jobs or min(len(sources), max(1, (os.cpu_count() or 4)))
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(_compile, sources))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed: {' '.join(cmd)}\n{res.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB} from {len(sources)} sources")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=None)
    build(ap.parse_args().jobs)
