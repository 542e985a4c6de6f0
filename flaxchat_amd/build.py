"""Build the gfx950 shared library `flaxchat_amd/libflaxchat_amd.so` in tree.

hipcc cross-compiles for gfx950 on a machine without a GPU. Packed-fp32
instruction selection is switched off for the device code.

    python -m flaxchat_amd.build
"""

from __future__ import annotations

import os
import re
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libflaxchat_amd.so")
ARCH = os.environ.get("FC_OFFLOAD_ARCH", "gfx950")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
SOURCES = ["fc_gemm.hip", "fc_attn.hip", "fc_forward.hip", "fc_sample.hip", "fc_paged.hip", "fc_tree.hip"]
FLAGS = [f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++17",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-I", os.path.join(HERE, "..", "include")]

# Sources none of whose kernels may spill scalar registers: the compiler has brought half of a spilled pointer back
# wrong there. Another compiler or an edit that makes one spill fails the build.
NO_SCALAR_SPILLS = ["fc_paged.hip", "fc_tree.hip"]


def check_scalar_spills(src: str, report: str):
    """Raises if the compiler's resource report names a kernel that spills scalar registers."""
    kernels = re.findall(r"Function Name: (\S+).*?SGPRs Spill: (\d+)", report, re.S)
    if not kernels:
        raise RuntimeError(f"no resource report for {src}:\n{report[-2000:]}")
    bad = [f"{k}: {n}" for k, n in kernels if int(n) > 0]
    if bad:
        raise RuntimeError(f"{src}: kernels that spill scalar registers: " + ", ".join(bad))


def _compile(src: str) -> str:
    obj = os.path.join(OBJ, os.path.splitext(src)[0] + ".o")
    watch = src in NO_SCALAR_SPILLS
    cmd = [HIPCC, *FLAGS, *(["-Rpass-analysis=kernel-resource-usage"] if watch else []), "-c",
           os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr[-6000:]}")
    if watch:
        check_scalar_spills(src, r.stderr)
    return obj


def build(verbose: bool = True) -> str:
    os.makedirs(OBJ, exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 1)) as ex:
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr[-6000:]}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    try:
        build()
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
