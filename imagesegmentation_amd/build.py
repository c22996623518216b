"""In-tree build of libisg.so for gfx950:  python -m imagesegmentation_amd.build [--force]"""
import glob
import os
import subprocess
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
OUT = os.path.join(_HERE, "libisg.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# (no packed float instructions: some forms of v_pk_*_f32, which -O3 makes of ordinary float code by itself, have given
# wrong results on this chip now and then; hipcc's host pass does not know the feature and says so, harmlessly)
NO_PACKED_F32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++20", "-fPIC", "-shared", "-Wall", "-Wno-unused-function"] + NO_PACKED_F32
# Per-file extras.  The fused backward is built without the SLP vectoriser: with it the gate arithmetic is laid out in
# register pairs, which costs ~30 vector registers (measured: -2 % on the 16-channel kernel, nothing lost on the others).
EXTRA_FLAGS = {"isg_convlstm_bwd.hip": ["-fno-slp-vectorize"]}


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def _stale():
    if not os.path.exists(OUT):
        return True
    # (this file as well: it holds the compiler's flags)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.h")) + [os.path.join(_HERE, "..", "include", "isg.h"),
                                                               os.path.abspath(__file__)]
    newest = max(os.path.getmtime(p) for p in deps)
    return os.path.getmtime(OUT) < newest


def build(force=False, verbose=True):
    """Compiles every csrc/*.hip into one shared object with hipcc (cross-compiles without a GPU)."""
    if not force and not _stale():
        return OUT
    objs = []
    procs = []
    objdir = os.path.join(_HERE, "csrc", "_obj")
    os.makedirs(objdir, exist_ok=True)
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        objs.append(obj)
        cmd = [HIPCC] + [f for f in FLAGS if f != "-shared"] + EXTRA_FLAGS.get(os.path.basename(src), []) + \
            ["-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd)))
    for src, p in procs:
        if p.wait() != 0:
            raise RuntimeError("hipcc failed on %s" % src)
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", OUT] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print("built", OUT)
