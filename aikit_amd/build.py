"""Build recipe for libenchip.so (gfx950) -- used by __graft_entry__.build().

Two translation units, compiled side by side by hipcc for gfx950 only and linked as a plain
C-ABI shared library next to this file. Flags that matter for correctness:

* ``-ffp-contract=off`` -- the epilogue must round after every multiply and add,
  as aikit's Go amd64 arithmetic does (no FMA contraction).
* ``-fhip-fp32-correctly-rounded-divide-sqrt`` -- the quantizer's maxAbs/127 and
  1/s and the erf tail's 1/(1+p*x) must be IEEE-correct divisions.
* ``-Xclang -target-feature -Xclang -packed-fp32-ops`` -- no packed-FP32 VALU ops
  (the host pass warns that it does not know the feature; harmless).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRCS = [os.path.join(HERE, "csrc", n) for n in ("enchip.hip", "attention_block.hip")]
OUT = os.path.join(HERE, "libenchip.so")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
]


def hipcc() -> str:
    p = os.path.join(ROCM, "bin", "hipcc")
    return p if os.path.exists(p) else (shutil.which("hipcc") or "hipcc")


def build(verbose: bool = False) -> str:
    """Compile libenchip.so in-tree; returns its path. Always recompiles."""
    tmp = OUT + ".tmp"
    inc = ["-I", os.path.join(ROOT, "include"), "-I", os.path.join(HERE, "csrc")]

    def check(cmd, proc):
        _, text = proc.communicate()
        noise = "'-packed-fp32-ops' is not a recognized feature"
        err = "\n".join(l for l in text.splitlines() if noise not in l)
        if proc.returncode != 0:
            raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{' '.join(cmd)}\n{err}")
        if verbose and err.strip():
            print(err)

    def start(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        return cmd, subprocess.Popen(cmd, stdout=subprocess.DEVNULL, stderr=subprocess.PIPE, text=True)

    with tempfile.TemporaryDirectory(prefix="enchip_build_") as d:
        objs = [os.path.join(d, os.path.basename(src) + ".o") for src in SRCS]
        running = [start([hipcc(), *HIPCC_FLAGS, *inc, "-c", src, "-o", o]) for src, o in zip(SRCS, objs)]
        try:
            for cmd, proc in running:
                check(cmd, proc)
        finally:
            for _, proc in running:
                if proc.poll() is None:
                    proc.kill()
                    proc.wait()
        check(*start([hipcc(), *HIPCC_FLAGS, "-shared", *objs, "-o", tmp, f"-Wl,-rpath,{ROCM}/lib"]))
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    print(build(verbose=True))
