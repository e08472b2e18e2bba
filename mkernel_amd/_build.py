"""Build libmk.so (gfx950 only) in-tree with hipcc.

The library is a plain C-ABI shared object (include/mk.h); nothing here links
against torch.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libmk.so"
SOURCES = ["mk_gemm.hip", "mk_gemm_small.hip", "mk_moe.hip", "mk_moe_index.hip", "mk_route.hip", "mk_w4.hip",
           "mk_product.hip", "mk_product_fwd.hip", "mk_product_grad.hip", "mk_probe.hip", "mk_capi.hip"]

HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    # packed-FP32 VALU forms stay disabled for every HIP translation unit
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found; libmk needs the ROCm toolchain to build")


def build(verbose: bool = False) -> Path:
    """Compile every HIP source and link mkernel_amd/libmk.so (always rebuilds).
    Sources are compiled side by side, at most 8 at once: one after another
    they take more than three minutes."""
    with tempfile.TemporaryDirectory() as d:
        objects = [str(Path(d) / (s + ".o")) for s in SOURCES]
        flags = [f for f in HIPCC_FLAGS if f != "-shared"]
        cmds = [[hipcc(), *flags, "-c", str(CSRC / s), "-o", o] for s, o in zip(SOURCES, objects)]
        with ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
            list(pool.map(_run, cmds))
        tmp = LIB.with_suffix(".so.tmp")
        cmds.append([hipcc(), *HIPCC_FLAGS, *objects, "-o", str(tmp)])
        _run(cmds[-1])
        if verbose:
            print("\n".join(" ".join(c) for c in cmds))
        os.replace(tmp, LIB)
    return LIB


def _run(cmd) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("libmk build failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)


if __name__ == "__main__":
    print(build(verbose=True))
