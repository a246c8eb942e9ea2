"""Build liboige_hip.so in-tree with hipcc for gfx950 (cross-compiles without a GPU).

    python -m omniisaacgymenvs_amd.build [--force]

-ffp-contract=off: the kernels spell out every fma the reference's torch ops perform
(oige_math.hpp) so fp32 rounding follows the reference; the compiler must not add more.
-packed-fp32-ops: no v_pk_add / mul / fma_f32; some of their forms have given wrong results on gfx950.
The sources are compiled side by side (one hipcc each) and linked: 82 s in one command, 28 s on 8 cores.
"""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "liboige_hip.so")
SOURCES = ["oige_core.hip", "locomotion.hip", "cartpole.hip", "hand.hip", "anymal_terrain.hip", "dr_noise.hip", "anymal.hip", "quadcopter.hip", "ball_balance.hip", "ingenuity.hip", "crazyflie.hip", "franka_cabinet.hip", "newhand_cabinet.hip", "observer.hip", "layer_norm.hip", "decay_attention.hip"]


def dependencies():
    """Every file the library is built from: all of csrc/ (*.hip, *.hpp) and include/*.h -- globbed, so a new header
    cannot be forgotten in the stale check."""
    import glob

    inc = os.path.join(HERE, "..", "include")
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.hpp"))
                  + glob.glob(os.path.join(inc, "*.h")))


FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-ffp-contract=off",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "hipcc"


def is_stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = dependencies() + [os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(out: str, defines=()) -> None:
    """Every source to an object (a few compilers at a time), then one link into ``out``."""
    jobs = max(1, min(8, int(os.environ.get("MAX_JOBS", 0) or os.cpu_count() or 1)))
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(jobs) as pool:
        objs = [os.path.join(tmp, os.path.splitext(s)[0] + ".o") for s in SOURCES]
        cmds = [[_hipcc()] + FLAGS + [f"-D{d}" for d in defines] + ["-c", os.path.join(CSRC, s), "-o", o]
                for s, o in zip(SOURCES, objs)]
        list(pool.map(subprocess.check_call, cmds))
        subprocess.check_call([_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC"] + objs + ["-o", out])


def build_variant(name: str, defines, verbose: bool = True) -> str:
    """Experiment builds: omniisaacgymenvs_amd/variants/liboige_<name>.so with extra -D flags (select with OIGE_LIB)."""
    out_dir = os.path.join(HERE, "variants")
    os.makedirs(out_dir, exist_ok=True)
    out = os.path.join(out_dir, f"liboige_{name}.so")
    if verbose:
        print("[oige build]", name, defines, flush=True)
    _compile(out, defines)
    return out


def build(force: bool = False, verbose: bool = True) -> str:
    if not force and not is_stale():
        return LIB
    if verbose:
        print("[oige build]", _hipcc(), " ".join(FLAGS), " ".join(SOURCES), "->", LIB, flush=True)
    _compile(LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
