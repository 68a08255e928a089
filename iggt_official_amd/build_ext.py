"""Build libiggt_hip.so (gfx950) in-tree with hipcc.  `python -m iggt_official_amd.build_ext`."""
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libiggt_hip.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=fast",
         "-Wno-unused-result", "-DNDEBUG",
         # no packed fp32 instructions (v_pk_add / mul / fma_f32): some of their forms have given wrong results on this hardware
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# extra flags of single translation units (measured choices, each explained in the file it applies to)
PER_FILE_FLAGS = {"attention_v3_est.hip": ["-mllvm", "-amdgpu-sched-strategy=max-ilp"]}


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def _stale(target, deps, cmd):
    """Missing, older than what it is made of, or made by another command line (kept beside it)."""
    if not os.path.exists(target) or not os.path.exists(target + ".cmd"):
        return True
    t = os.path.getmtime(target)
    with open(target + ".cmd") as f:
        return f.read() != " ".join(cmd) or any(os.path.getmtime(d) > t for d in deps)


def _start(target, cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    if os.path.exists(target + ".cmd"):
        os.remove(target + ".cmd")
    return target, cmd, subprocess.Popen(cmd)


def _finish(target, cmd, process):
    if process.wait() != 0:
        raise RuntimeError(f"hipcc failed on {target}")
    with open(target + ".cmd", "w") as f:
        f.write(" ".join(cmd))


def build(force=False, verbose=True):
    os.makedirs(LIB_DIR, exist_ok=True)
    obj_dir = os.path.join(LIB_DIR, "obj")
    os.makedirs(obj_dir, exist_ok=True)
    headers = glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    headers.append(os.path.join(CSRC, "attention_v3.hip"))   # included by attention_v3_est.hip
    objs, jobs = [], []
    for src in sources():
        obj = os.path.join(obj_dir, os.path.basename(src)[:-4] + ".o")
        objs.append(obj)
        cmd = [HIPCC] + FLAGS + PER_FILE_FLAGS.get(os.path.basename(src), []) + ["-c", src, "-o", obj]
        if force or _stale(obj, [src] + headers, cmd):
            jobs.append(_start(obj, cmd, verbose))
    failed = []
    for job in jobs:
        try:
            _finish(*job)
        except RuntimeError as e:
            failed.append(str(e))
    if failed:
        raise RuntimeError("; ".join(failed))
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
    if force or jobs or _stale(LIB, objs, cmd):
        _finish(*_start(LIB, cmd, verbose))
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
