"""Builds libsage_hip.so (the gfx950 SageAttention2 forward path) in-tree.

    python sota-papers-lab_amd/build.py

Compiles every source under csrc/ with hipcc for gfx950 and links
spl_sage/libsage_hip.so next to the Python mirror of the API. Objects go to
_build/ (git-ignored). Packed FP32 instructions are disabled for all device
code; the prologue and the rotary and cache writes are compiled with
-ffp-contract=off so their fp32 arithmetic is exactly the written operation
order, and the attention source twice (see UNITS).
"""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = PKG / "_build"
LIB = PKG / "spl_sage" / "libsage_hip.so"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

COMMON = [
    "-O3",
    "-std=c++17",
    "-fPIC",
    f"--offload-arch={ARCH}",
    "-Wall",
    "-Wno-unused-function",
    # No packed fp32 (v_pk_fma_f32, v_pk_mul_f32, v_pk_add_f32) anywhere: on the
    # MI355X machines this library is tested on, some of their forms have given
    # wrong results now and then without an error.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]
SCHED = ["-mllvm", "--amdgpu-sched-strategy=iterative-maxocc", "-mllvm", "--misched-postra-direction=bottomup"]
# (source, object, extra flags). The attention source is compiled twice: its
# dense and causal kernels with LLVM's occupancy-keeping iterative pre-RA
# scheduler and a bottom-up post-RA pass (SCHED: instruction order only,
# outputs bit-identical, 1.5-2.4% faster at C2-C5), its merged kernels
# (SAGE_ATTN_MERGED) with the default order, which is faster for them.
UNITS = [
    ("sage_prologue.hip", "sage_prologue.hip.o", ["-ffp-contract=off"]),
    ("sage_attention.hip", "sage_attention.hip.o", SCHED),
    ("sage_attention.hip", "sage_attention_merged.hip.o", ["-DSAGE_ATTN_MERGED"]),
    ("sage_attn_keys.hip", "sage_attn_keys.hip.o", []),
    ("sage_peak.hip", "sage_peak.hip.o", []),
    ("sage_noalloc.hip", "sage_noalloc.hip.o", []),
    ("sage_cache.hip", "sage_cache.hip.o", ["-ffp-contract=off"]),
    ("sage_cache_attn.hip", "sage_cache_attn.hip.o", []),
    ("sage_api.cpp", "sage_api.cpp.o", []),
    ("sage_cache_api.cpp", "sage_cache_api.cpp.o", []),
]


def _run(cmd, what: str) -> str:
    """Runs one step; returns what it wrote to stderr. A failure names the step,
    its exit status (a compiler killed from outside writes nothing) and its
    command."""
    res = subprocess.run(cmd, capture_output=True, text=True, errors="replace")
    # hipcc's host pass does not know the packed-fp32 feature and says so; that is harmless.
    noise = "'-packed-fp32-ops' is not a recognized feature"
    err = "\n".join(l for l in res.stderr.splitlines() if noise not in l)
    if res.returncode != 0:
        how = f"killed by signal {-res.returncode}" if res.returncode < 0 else f"exit status {res.returncode}"
        raise RuntimeError(f"{what} failed ({how}): {' '.join(cmd)}\n{res.stdout}{err}")
    return err


def _compile(unit) -> Path:
    src, obj, extra = unit
    out = OBJ / obj
    lang = ["-x", "hip"] if src.endswith(".hip") else []
    err = _run([HIPCC, *COMMON, *extra, *lang, "-c", str(CSRC / src), "-o", str(out)], f"compiling {obj}")
    if err.strip():
        print(err, file=sys.stderr)
    return out


def build(verbose: bool = True) -> Path:
    """Compile and link; returns the library path. Raises on failure."""
    OBJ.mkdir(exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(6, len(UNITS))) as ex:
        objs = list(ex.map(_compile, UNITS))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [HIPCC, "-shared", f"--offload-arch={ARCH}", "-fPIC", *map(str, objs), "-o", str(tmp)]
    _run(cmd, f"linking {LIB.name}")
    # Every kernel the launchers name must be in the library: load it with all
    # symbols resolved now (a kernel the host pass failed to instantiate shows
    # up here, not at first use on a GPU box).
    try:
        ctypes.CDLL(str(tmp), mode=os.RTLD_NOW)
    except OSError as e:
        raise RuntimeError(f"built library does not load: {e}") from e
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build()
