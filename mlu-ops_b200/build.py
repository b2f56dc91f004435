"""Builds libmluops_b200.so: the C-ABI library with the sm_100a kernels.

One nvcc invocation for each C++ host source and CUDA file, then one that links
them; the output is placed next to this file under lib/ (git-ignored, shipped as
a built artefact).  nvcc cross-compiles, so no GPU is needed to build.

Usage: python mlu-ops_b200/build.py [--force] [--verbose]
"""
import concurrent.futures
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
OBJ_DIR = os.path.join(LIB_DIR, "obj")
LIB = os.path.join(LIB_DIR, "libmluops_b200.so")


KERNEL_DIRS = ("sparse_conv", "voxelization", "dynamic_point_to_voxel", "multi_tensor_adamw", "group_norm_act",
               "grouped_matmul")


def sources():
    out = sorted(glob.glob(os.path.join(CSRC, "core", "*.cpp")))
    for d in KERNEL_DIRS:
        for pattern in ("*.cpp", "*.cu"):
            out += sorted(glob.glob(os.path.join(CSRC, "kernels", d, pattern)))
    return out


def headers():
    out = (glob.glob(os.path.join(ROOT, "include", "*.h")) + glob.glob(os.path.join(CSRC, "core", "*.h"))
           + glob.glob(os.path.join(CSRC, "core", "*.cuh")))
    for d in KERNEL_DIRS:
        for pattern in ("*.h", "*.cuh"):
            out += glob.glob(os.path.join(CSRC, "kernels", d, pattern))
    return out


def up_to_date():
    if not os.path.isfile(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= t for p in sources() + headers() + [os.path.abspath(__file__)])


def build(force=False, verbose=False):
    if not force and up_to_date():
        return LIB
    os.makedirs(OBJ_DIR, exist_ok=True)
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    flags = [
        "-std=c++17", "-O3", "-lineinfo",
        "-gencode", "arch=compute_100a,code=sm_100a",
        "-Xcompiler", "-fPIC,-fvisibility=hidden,-Wall",
        "-DMLUOP_WIN_API=__attribute__((visibility(\"default\")))",
        "-x", "cu",
        "-I", os.path.join(ROOT, "include"), "-I", CSRC,
    ]
    if verbose:
        flags += ["-Xptxas", "-v"]
    flags += os.environ.get("MLUOP_B200_NVCC_FLAGS", "").split()  # extra compiler flags (experiments)

    # One object per source, compiled side by side; an object is kept while its own source, every
    # header and the flags are older than it.  What a build that fails or is cut off leaves behind is
    # not taken for more: outputs get their names when they are whole, and the flags' file says
    # nothing while objects of other flags come in.
    flag_file = os.path.join(OBJ_DIR, "flags.txt")
    same_flags = os.path.isfile(flag_file) and open(flag_file).read() == " ".join([nvcc] + flags)
    if not same_flags and os.path.isfile(flag_file):
        os.remove(flag_file)
    newest_header = max(os.path.getmtime(p) for p in headers())

    def run(out, cmd):
        part = os.path.join(os.path.dirname(out), "part." + os.path.basename(out))
        subprocess.check_call([nvcc, "-o", part] + cmd)
        os.replace(part, out)

    def compile_one(src):
        obj = os.path.join(OBJ_DIR, os.path.relpath(src, CSRC).replace(os.sep, "__") + ".o")
        if (force or not same_flags or not os.path.isfile(obj)
                or os.path.getmtime(obj) < max(os.path.getmtime(src), newest_header)):
            cmd = ["-c"] + flags + [src]
            if verbose:
                print(" ".join([nvcc] + cmd))
            run(obj, cmd)
        return obj

    with concurrent.futures.ThreadPoolExecutor(os.cpu_count()) as pool:
        objects = list(pool.map(compile_one, sources()))
    with open(flag_file, "w") as f:
        f.write(" ".join([nvcc] + flags))
    run(LIB, ["-shared", "-gencode", "arch=compute_100a,code=sm_100a"] + objects
        + ["-lcudart_static", "-lpthread", "-ldl", "-lrt"])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
