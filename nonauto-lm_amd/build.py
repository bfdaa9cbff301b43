"""In-tree build of libmivae.so (hand-written HIP kernels + C ABI) for gfx950.

hipcc cross-compiles without a GPU; the .so is git-ignored but travels with the gpurun snapshot.
Usage:  python nonauto-lm_amd/build.py [--force]
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libmivae.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
RECIPE = os.path.abspath(__file__)       # an object compiled with other flags is out of date like one of another source
SOURCES = ["elementwise.hip", "nice_stack.hip", "nice_small.hip", "nice_big.hip", "invlinear.hip", "pairwise.hip", "mixed_stack.hip", "attention.hip", "biased_attention.hip", "token_attention.hip", "qk_rotary.hip", "nll.hip", "optim.hip", "layernorm.hip", "linear.hip", "maf.hip"]
# packed-fp32-ops off: hipcc -O3 otherwise forms v_pk_{add,mul,fma}_f32 from ordinary float code, and some operand forms
# of these have been seen to return wrong values now and then.  (The host pass warns that it does not know the feature.)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fno-gpu-rdc",
         "-Wno-unused-result", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# The MFMA kernels keep their f32 VALU work single-issue: beside MFMAs a packed v_pk_*_f32 costs more than the two plain
# instructions it replaces (MI355X_MICROARCH.md, "price of one filler beside MFMAs").
EXTRA_FLAGS = {"nice_big.hip": ["-fno-slp-vectorize"], "nll.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"]}


def _newer(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=True):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    os.makedirs(LIBDIR, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hpp")]
    abi = os.path.join(INCLUDE, "mivae.h")         # included by the sources whose entry points take its structs
    srcs = [os.path.join(CSRC, s) for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    objs = [os.path.join(LIBDIR, os.path.basename(s)[:-4] + ".o") for s in srcs]

    def compile_one(pair):
        src, obj = pair
        with open(src) as f:
            deps = [src, RECIPE] + headers + ([abi] if '"mivae.h"' in f.read() else [])
        if force or _newer(obj, deps):
            cmd = [hipcc] + FLAGS + ["-I", INCLUDE] + EXTRA_FLAGS.get(os.path.basename(src), []) + ["-c", src, "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.check_call(cmd)
            return True
        return False

    with ThreadPoolExecutor(max_workers=4) as ex:
        rebuilt = list(ex.map(compile_one, zip(srcs, objs)))
    if force or any(rebuilt) or _newer(LIB, objs):
        cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
