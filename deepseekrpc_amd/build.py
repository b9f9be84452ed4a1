"""Build ``libdsr_sampling.so`` in-tree with hipcc for gfx950.

    python -m deepseekrpc_amd.build [source ...]

Flags that the numerics depend on:
  -ffp-contract=off   no FMA contraction: the penalty, scaling and ratio
                      arithmetic must round like the reference's NumPy float64
                      (its own CUDA build passes --fmad=false, native/setup.py:19);
  no -ffast-math      IEEE division and float64 denormals are required
                      (temperature 1e-320 is a tested input).
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OUT = os.path.join(HERE, "libdsr_sampling.so")
# Each source is one object; their kernels share no device symbols.
SOURCES = {
    "dsr_sampling.hip": ["dsr_common.h", "dsr_wave.h", "dsr_general.h", "dsr_fast.h", "dsr_topk.h", "dsr_full.h",
                         "dsr_verify.h", "dsr_history.h", "dsr_split.h", "dsr_numpy.h", "dsr_head.h", "dsr_f32.h",
                         "dsr_wide.h", "dsr_wide_verify.h"],
    "dsr_tree.hip": ["dsr_plan.h", "dsr_rotary.h", "dsr_attention.h", "dsr_attention_wide.h",
                     "dsr_commit.h"],
    "dsr_branch.hip": ["dsr_beams.h", "dsr_pages.h"],
    "dsr_prefix.hip": ["dsr_prefix.h", "dsr_attention.h", "dsr_attention_wide.h"],
}

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
    # Packed FP32 instructions stay off (they are not needed on this path).
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _run(cmds, verbose):
    """Run the compiler commands side by side; raise on the first that failed."""
    procs = [subprocess.Popen(cmd, stdout=subprocess.DEVNULL, stderr=subprocess.PIPE, text=True) for cmd in cmds]
    errors = [proc.communicate()[1] for proc in procs]
    noise = "is not a recognized feature for this target"
    for proc, text in zip(procs, errors):
        err = "\n".join(line for line in text.splitlines() if noise not in line)
        if proc.returncode != 0:
            raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{err}")
        if verbose and err.strip():
            print(err, file=sys.stderr)


def build(verbose: bool = False, only=None) -> str:
    """Compile every source (or the named ones, with the others' objects from
    an earlier build) and link the library."""
    objects = {s: os.path.join(CSRC, s.replace(".hip", ".o")) for s in SOURCES}
    todo = [s for s in SOURCES if only is None or s in only or not os.path.exists(objects[s])]
    _run([[HIPCC, *FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", os.path.join(CSRC, s), "-o", objects[s]] for s in todo],
         verbose)
    _run([[HIPCC, "--offload-arch=gfx950", "-shared", *objects.values(), "-o", OUT + ".tmp"]], verbose)
    os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(verbose=True, only=sys.argv[1:] or None))
