"""Builds libaesir_hip.so for gfx950 with hipcc (cross-compiles; no GPU needed).

    python runeforgeai-project-aesir_amd/build.py [--jobs N]

Objects go to runeforgeai-project-aesir_amd/_build/, the library to
runeforgeai-project-aesir_amd/aesir_hip/libaesir_hip.so (loaded by aesir_hip/__init__.py).
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "aesir_hip", "libaesir_hip.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

CXXFLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # f16 rounding points must survive compilation: no multiply-add contraction anywhere
    "-ffp-contract=off",
    # keep the compiler from emitting packed-FP32 VALU ops
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-variable", "-Wno-unused-function", "-Wno-unused-result",
    f"-I{os.path.join(REPO, 'include')}",
    f"-I{CSRC}",
]

SOURCES = ["ctx.hip", "gemv.hip", "quant.hip", "skinny.hip", "skinny_raw.hip", "attention.hip", "kv4.hip", "basic.hip", "q8_0.hip", "abi_ops.hip", "model.hip",
           "prefill.hip", "gguf.hip", "sampler.hip", "blas.hip"]


# accumulators of the matrix instructions in vector registers: kernels that rescale them each time a maximum rises
# would otherwise move them from the accumulation registers and back
EXTRA = {"kv4.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]}


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.splitext(src)[0] + ".o")
    cmd = [HIPCC, *CXXFLAGS, *EXTRA.get(src, []), "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in r.stderr.splitlines() if noise not in l)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{err}")
    if err.strip():
        sys.stderr.write(err + "\n")
    return obj


def build(jobs: int | None = None) -> str:
    os.makedirs(BUILD, exist_ok=True)
    jobs = jobs or min(8, os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(jobs) as ex:
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    # hipBLASLt for the prefill GEMMs of long chunks (blas.hip)
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs, "-L/opt/rocm/lib", "-lhipblaslt",
           "-Wl,-rpath,/opt/rocm/lib"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=None)
    print(build(ap.parse_args().jobs))
