"""Builds libhelrm_hip.so (gfx950) in-tree with hipcc.

    python -m helrm_amd.build

The library goes to helrm_amd/_lib/libhelrm_hip.so so that it ships with the
source tree; nothing is installed into site-packages.
"""
import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
LIB = os.path.join(OUT_DIR, "libhelrm_hip.so")
SOURCES = ["kernels.hip", "ntt.hip", "encoder.hip", "runtime.hip", "norm.hip", "products.hip", "skinny.hip",
           "cleartext.hip"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # float64 encoder/decoder arithmetic must not be contracted into FMAs
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # matrix instructions on ordinary registers: with accumulation registers the compiler moves the sums to and fro
    "-mllvm", "-amdgpu-mfma-vgpr-form",
]


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("hipcc failed building libhelrm_hip.so")


def build(verbose=False):
    """Compiles every source, each in a process of its own, and links them."""
    os.makedirs(OUT_DIR, exist_ok=True)
    tmp = LIB + ".tmp"
    with tempfile.TemporaryDirectory() as d, ThreadPoolExecutor(len(SOURCES)) as pool:
        objs = [os.path.join(d, s + ".o") for s in SOURCES]
        list(pool.map(lambda so: _run([HIPCC] + FLAGS + ["-c", os.path.join(CSRC, so[0]), "-o", so[1]], verbose), zip(SOURCES, objs)))
        _run([HIPCC, "--offload-arch=gfx950", "-shared"] + objs + ["-o", tmp], verbose)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
