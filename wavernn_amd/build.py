"""Build libwrnn_mi355.so in-tree with hipcc for gfx950 (cross-compiles without a GPU).

One object per source under lib/obj/ (recompiled only when the source, a header or this file changed, several at a
time), then one link: editing one kernel file costs one file's compile."""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
OBJ_DIR = os.path.join(LIB_DIR, "obj")
LIB_PATH = os.path.join(LIB_DIR, "libwrnn_mi355.so")
SOURCES = ["taco_decoder.hip", "length_regulator.hip", "bilstm.hip", "bigru.hip", "durations.hip", "wavernn.hip",
           "aligner.hip", "mol.hip", "relative_bias.hip", "attention.hip"] + [
               f"attention_{d}_{t}.hip" for d in ("forward", "backward") for t in ("bf16", "bf16_d256", "f32", "f32_d256")]
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function"]
# The attention kernels are built without packed fp32 instructions: some of their forms have given wrong results on this
# hardware, with no error.  (The host pass does not know the feature and says so; harmless.)  The older kernels keep the code they were
# verified with: the teacher-forced loop loses 5.5 % without them (13.7 -> 14.5 us per decoder step at B=64).
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# MFMA_IN_VGPRS: sums stay in the vector registers that the softmax works on; by default every value that passes between
# matrix and vector instructions is copied.  2 x 16 heads, 2048 x 2048 in float32 at 128 columns: 376 -> 366 us; bfloat16 at 256
# columns, 2 x 8 heads, 4096 x 4096: 796 -> 419 us.  The bfloat16 backward pass at 64 and 128 columns is the slower for it (551 -> 467 TFLOP/s).
MFMA_IN_VGPRS = ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]
SOURCE_FLAGS = {s: NO_PACKED_FP32 + (MFMA_IN_VGPRS if s in ("attention_forward_bf16_d256.hip", "attention_forward_f32.hip",
                                                            "attention_forward_f32_d256.hip", "attention_backward_bf16_d256.hip",
                                                            "attention_backward_f32.hip", "attention_backward_f32_d256.hip") else [])
                for s in SOURCES if s.startswith(("attention", "relative_bias"))}


def _hipcc() -> str:
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    return "hipcc"


def _shared():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    hs.append(os.path.join(HERE, "..", "include", "wrnn_mi355.h"))
    hs.append(__file__)     # the flags
    return hs


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def needs_build() -> bool:
    deps = [os.path.join(CSRC, s) for s in SOURCES] + _shared()
    return _stale(LIB_PATH, deps)


def build(force: bool = False, verbose: bool = True) -> str:
    if not force and not needs_build():
        return LIB_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    shared = _shared()
    jobs = []
    for s in SOURCES:
        src, obj = os.path.join(CSRC, s), os.path.join(OBJ_DIR, s[:-4] + ".o")
        if force or _stale(obj, [src] + shared):
            jobs.append([_hipcc()] + FLAGS + SOURCE_FLAGS.get(s, []) + ["-c", src, "-o", obj])

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)

    workers = max(1, min(len(jobs), int(os.environ.get("MAX_JOBS", "0")) or (os.cpu_count() or 4), 8))
    with ThreadPoolExecutor(workers) as ex:
        list(ex.map(run, jobs))
    objs = [os.path.join(OBJ_DIR, s[:-4] + ".o") for s in SOURCES]
    run([_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB_PATH] + objs)
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB_PATH)
