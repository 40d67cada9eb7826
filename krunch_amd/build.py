"""Build libkrunch_hip.so (gfx950) in-tree with hipcc.

    python -m krunch_amd.build            # or krunch_amd.build.build()

Objects go to krunch_amd/_build/, the library to krunch_amd/libkrunch_hip.so.
Every file is compiled with -ffp-contract=off (bit-identical packed and
stepped numerics) and with packed-fp32 instructions disabled.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT_DIR = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libkrunch_hip.so")
ARCH = os.environ.get("KRUNCH_OFFLOAD_ARCH", "gfx950")

SOURCES = ["kr_rc.hip", "kr_cdf.hip", "kr_gemm.hip", "kr_quant.hip", "kr_layer.hip", "kr_engine.hip",
           "kr_wide.hip", "kr_mid.hip", "kr_wkv.hip",
           "kr_step.hip", "kr_head.hip", "kr_pack.hip", "kr_scores.hip", "kr_w4.hip", "kr_heads.hip",
           "kr_headloss.hip", "kr_delta.hip"]

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wall", "-Wno-unused-function", "-I", CSRC, "-I", INCLUDE]


def _compile(src: str) -> str:
    obj = os.path.join(OUT_DIR, os.path.splitext(src)[0] + ".o")
    cmd = [HIPCC, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def build(verbose: bool = False) -> str:
    os.makedirs(OUT_DIR, exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(8, len(SOURCES))) as ex:
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print("built", LIB)
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
