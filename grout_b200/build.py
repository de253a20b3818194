"""Builds libgrout_attn.so in-tree with nvcc for sm_100a.

    python -m grout_b200.build [--force]

One object per .cu file under csrc/, linked into grout_b200/libgrout_attn.so
(static CUDA runtime, so the library carries no dependency beyond the
driver).  The Python binding csrc/bind.cpp becomes bind_path() (g++, PyTorch's
headers), a file for each PyTorch and Python that it is built for: its compiled
code holds their object layouts.  The library does not need it, and is there
without it where PyTorch is missing or the binding does not compile.  Each is
built where it is missing or older than one of its sources.
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


def bind_path() -> str:
    """The binding's file for this PyTorch and Python."""
    import torch  # only its version is needed

    return os.path.join(HERE, f"_bind.torch-{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX')}")


def _newer(path: str, deps) -> bool:
    return os.path.exists(path) and all(os.path.getmtime(p) <= os.path.getmtime(path) for p in deps)


def _lib_up_to_date() -> bool:
    return _newer(LIB, _sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + [
        os.path.join(ROOT, "include", "grout_attn.h"), __file__])


def _bind_up_to_date() -> bool:
    return _newer(bind_path(), [os.path.join(CSRC, "bind.cpp"), os.path.join(ROOT, "include", "grout_attn.h"), __file__])


def up_to_date() -> bool:
    return _lib_up_to_date() and _bind_up_to_date()


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


def _compile(commands) -> None:
    """Runs the compilers side by side and waits for all of them."""
    procs = [(subprocess.Popen(cmd), cmd) for cmd in commands]
    failed = [cmd for p, cmd in procs if p.wait() != 0]
    if failed:
        raise RuntimeError("compilation failed: " + "; ".join(" ".join(cmd) for cmd in failed))


def _build_lib(verbose: bool, extra_flags) -> None:
    os.makedirs(BUILD_DIR, exist_ok=True)
    objs = [os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o") for src in _sources()]
    commands = [[nvcc(), *NVCC_FLAGS, *extra_flags, "-c", src, "-o", obj] for src, obj in zip(_sources(), objs)]
    if verbose:
        for cmd in commands:
            print(" ".join(cmd))
    _compile(commands)
    tmp = LIB + ".tmp"
    _compile([[nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", tmp, *objs]])
    os.replace(tmp, LIB)


def _build_bind(verbose: bool) -> None:
    tmp = bind_path() + ".tmp"
    cmd = _bind_command(tmp)
    if verbose:
        print(" ".join(cmd))
    _compile([cmd])
    os.replace(tmp, bind_path())


def build(force: bool = False, verbose: bool = False, extra_flags=()) -> str:
    if force or not _lib_up_to_date():
        _build_lib(verbose, extra_flags)
    try:
        if force or not _bind_up_to_date():
            _build_bind(verbose)
    except ImportError as e:  # no PyTorch: nobody to call the binding
        print(f"grout_b200: the Python binding is not built: {e}", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    v = "-v" in sys.argv
    extra = ["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else []
    print(build(force="--force" in sys.argv or bool(extra), verbose=v, extra_flags=extra))
