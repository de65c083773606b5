"""In-tree build of libhh.so (hand-written gfx950 HIP kernels + C ABI).

    python -m helping_hand_for_egocentric_videos_amd.build [--force]

hipcc cross-compiles for gfx950 without a GPU; the resulting .so is git-ignored but travels with
the tree to the GPU box.  Objects are cached under csrc/_obj keyed by source mtime.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "_obj")
LIB = os.path.join(HERE, "libhh.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# no packed fp32 instructions (v_pk_add / mul / fma_f32): the compiler forms them from ordinary float code, and some of their operand forms have
# given wrong results on this hardware; the same arithmetic as scalar instructions has not.  It costs the training step about 1 % (295.2 -> 292.4 clips/s).  (The host pass does not know the feature and says so.)
FLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-Wno-unused-result", "-Wno-unused-value",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# per-file additions.  attn_space32.hip: its fully unrolled chunk loops trip -Wpass-failed (a `#pragma unroll 1` loop of the rare redo path)
EXTRA_FLAGS = {"attn_space32.hip": ["-Wno-pass-failed", "-Wno-inline-asm"]}


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".hip") or f.endswith(".cpp"))


def _newer(a, b):
    return not os.path.exists(b) or os.path.getmtime(a) > os.path.getmtime(b)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    hdr = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")] + [os.path.join(HERE, "..", "include", "hh.h")]
    hdr_m = max(os.path.getmtime(h) for h in hdr)
    jobs = []
    for src in sources():
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ, src + ".o")
        if force or _newer(s, o) or os.path.getmtime(o) < hdr_m:
            cmd = [HIPCC] + FLAGS + EXTRA_FLAGS.get(src, []) + (["-x", "hip"] if src.endswith(".cpp") else []) + ["-c", s, "-o", o]
            jobs.append(cmd)

    def run(cmd):
        if verbose:
            print(" ".join(cmd))
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("hipcc failed:\n%s\n%s" % (" ".join(cmd), r.stderr))
        return r.stderr

    if jobs:
        with ThreadPoolExecutor(max_workers=min(6, len(jobs))) as ex:
            list(ex.map(run, jobs))
    objs = [os.path.join(OBJ, s + ".o") for s in sources()]
    if jobs or not os.path.exists(LIB) or any(_newer(o, LIB) for o in objs):
        run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
