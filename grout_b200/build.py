"""Builds libgrout_attn.so in-tree with nvcc for sm_100a.

    python -m grout_b200.build [--force]

One object per .cu file under csrc/, linked into grout_b200/libgrout_attn.so
(static CUDA runtime, so the library carries no dependency beyond the
driver).  The Python binding csrc/bind.cpp becomes
grout_b200/_bind.so (g++, PyTorch's headers).  The build is skipped when both are
newer than every source.
"""
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libgrout_attn.so")
BIND = os.path.join(HERE, "_bind.so")
BUILD_DIR = os.path.join(HERE, "_build")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-I" + os.path.join(ROOT, "include"),
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps():
    return _sources() + [os.path.join(CSRC, "bind.cpp")] + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(
        os.path.join(CSRC, "*.h")) + [os.path.join(ROOT, "include", "grout_attn.h"), __file__]


def up_to_date() -> bool:
    if not (os.path.exists(LIB) and os.path.exists(BIND)):
        return False
    t = min(os.path.getmtime(LIB), os.path.getmtime(BIND))
    return all(os.path.getmtime(p) <= t for p in _deps())


def _bind_command(out: str):
    import torch  # only its paths are needed

    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    include = [os.path.join(ROOT, "include"), sysconfig.get_paths()["include"], os.path.join(root, "include"),
               os.path.join(root, "include", "torch", "csrc", "api", "include"), os.path.join(cuda, "include")]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *("-I" + d for d in include),
            os.path.join(CSRC, "bind.cpp"), "-o", out, "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda",
            "-ltorch_cpu", "-ltorch_python"]


def build(force: bool = False, verbose: bool = False, extra_flags=()) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(BUILD_DIR, exist_ok=True)
    objs = []
    procs = []
    for src in _sources():
        obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o")
        cmd = [nvcc(), *NVCC_FLAGS, *extra_flags, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        procs.append((subprocess.Popen(cmd), cmd))
        objs.append(obj)
    cmd = _bind_command(BIND + ".tmp")
    procs.append((subprocess.Popen(cmd), cmd))
    for p, cmd in procs:
        if p.wait() != 0:
            raise RuntimeError("compilation failed: " + " ".join(cmd))
    os.replace(BIND + ".tmp", BIND)
    tmp = LIB + ".tmp"
    cmd = [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", tmp, *objs]
    subprocess.check_call(cmd)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    v = "-v" in sys.argv
    extra = ["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else []
    print(build(force="--force" in sys.argv or bool(extra), verbose=v, extra_flags=extra))
