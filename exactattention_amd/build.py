"""Builds libexactattn_hip.so in-tree with hipcc for gfx950 (python -m exactattention_amd.build)."""

from __future__ import annotations

import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

SOURCES = ["ea_hip.hip", "ea_decode.hip", "ea_mrow.hip", "ea_four.hip", "ea_prefill.hip", "ea_prefill_mod.hip",
           "ea_step.hip", "ea_norm.hip", "ea_draft.hip", "ea_exact_host.cpp", "ea_csr.cpp"]
HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libexactattn_hip.so")

# -packed-fp32-ops: never emit packed fp32 VALU ops (some of their forms have given wrong results).
# -fno-gpu-flush-denormals-to-zero: bf16 subnormals convert exactly through fp32.
# -amdgpu-mfma-vgpr-form=1: MFMA operands and accumulators in VGPRs; the prefill kernel's int32
#  accumulators are also read by VALU folds, and the AGPR file then serves as cheap spill space
#  (the AGPR form spills the kernel's working set to scratch).
HIPCC_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
               "-fno-gpu-flush-denormals-to-zero", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
               "-mllvm", "-amdgpu-mfma-vgpr-form=1", "-Wall", "-Wno-unused-function"]
# and for one source alone; the reason stands there
FILE_FLAGS = {f: ["-mllvm", "-disable-machine-licm=1"] for f in ("ea_prefill_mod.hip", "ea_four.hip")}


def build(verbose: bool = False) -> str:
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    gen = os.path.join(CSRC, "gen_tables.py")
    subprocess.run([sys.executable, gen], check=True, stdout=subprocess.DEVNULL)
    tmp = LIB + ".tmp"
    with tempfile.TemporaryDirectory() as objs:
        def run(cmd):
            return subprocess.run([hipcc, *cmd], capture_output=True, text=True)

        out = [os.path.join(objs, f + ".o") for f in SOURCES]
        with ThreadPoolExecutor(8) as pool:
            done = list(pool.map(lambda x: run([*HIPCC_FLAGS, *FILE_FLAGS.get(x[0], []), "-c", os.path.join(CSRC, x[0]), "-o", x[1]]),
                                 zip(SOURCES, out)))
        if all(r.returncode == 0 for r in done):
            done.append(run(["--offload-arch=gfx950", "-shared", "-o", tmp, *out]))
        for r in done:
            if r.returncode != 0:
                sys.stderr.write(r.stdout + r.stderr)
                raise RuntimeError("hipcc failed building libexactattn_hip.so")
            if verbose:
                sys.stderr.write(r.stderr)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
