"""Build librstr_hip.so for gfx950 in-tree (pretrained-rstr_amd/lib/).

hipcc flags: -ffp-contract=off (every fused multiply-add is written explicitly;
the CPU restatement relies on it), and packed FP32 instructions disabled.
"""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "lib", "librstr_hip.so")

HIP_SOURCES = ["kernels.hip", "kv4.hip", "step_ops.hip", "pool_attn.hip", "pool_rows.hip", "rstr_hip.cpp", "device_ops.cpp",
               "pool_ops.cpp"]
HIPCC_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
               "-ffp-contract=off", "-Wno-unused-value",
               "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


HIPCC = ["hipcc", *HIPCC_FLAGS]


def _check(stderr: str, code: int):
    noise = "is not a recognized feature for this target"
    if code != 0:
        raise RuntimeError(f"hipcc failed ({code}):\n" + "\n".join(l for l in stderr.splitlines() if noise not in l))


def build(verbose: bool = False) -> str:
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    with tempfile.TemporaryDirectory(prefix="rstr_build_") as tmp:  # one compiler a source, side by side
        objs = [os.path.join(tmp, s + ".o") for s in HIP_SOURCES]
        jobs = [[*HIPCC, "-c", os.path.join(CSRC, s), "-o", o] for s, o in zip(HIP_SOURCES, objs)]
        procs = [subprocess.Popen(c, stdout=subprocess.DEVNULL, stderr=subprocess.PIPE, text=True) for c in jobs]
        for cmd, p in zip(jobs, procs):
            if verbose:
                print(" ".join(cmd), flush=True)
            _check(p.communicate()[1], p.returncode)
        r = subprocess.run([*HIPCC, "-shared", *objs, "-o", OUT + ".tmp"], capture_output=True, text=True)
        _check(r.stderr, r.returncode)
    os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
