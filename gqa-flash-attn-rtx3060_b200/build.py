"""Builds libgqa_sm100.so (the C-ABI library) in-tree for sm_100a, and the serving step's
Python binding (_serving_ext.so, host code against torch's headers). The library needs
nvcc alone; the binding, which only Python callers use, is left out without torch or g++.

    python gqa-flash-attn-rtx3060_b200/build.py [--force] [--debug]

The library is one translation unit (csrc/gqa_sm100.cu) compiled by nvcc with
`-gencode arch=compute_100a,code=sm_100a` and the static CUDA runtime; it does
not link libcuda (the driver's tensor-map encoder is looked up at run time),
so it loads on a machine without a GPU driver.
"""
import argparse
import contextlib
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import uuid

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT = os.path.join(HERE, "gqa_kernels", "libgqa_sm100.so")
# Debug variant: in-kernel address/coordinate checks (GQA_DEBUG_CHECKS) that report
# GQA_ERR_DEBUG_CHECK instead of faulting; selected at run time with
# GQA_KERNELS_LIB=debug.
OUT_DEBUG = os.path.join(HERE, "gqa_kernels", "libgqa_sm100_debug.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "-cudart", "static",
]


EXT = os.path.join(HERE, "gqa_kernels", "_serving_ext.so")
EXT_SOURCES = [os.path.join(CSRC, "serving_ext.cpp"), os.path.join(INCLUDE, "gqa_sm100.h")]


@contextlib.contextmanager
def _written(out):
    """A path of its own to write, put in `out`'s place at the end: builds may run at the same time."""
    tmp = f"{out}.{uuid.uuid4().hex}.tmp"
    try:
        yield tmp
        os.replace(tmp, out)
    finally:
        if os.path.exists(tmp):
            os.remove(tmp)


def build_ext(force=False):
    """Compiles gqa_kernels._serving_ext (g++, a few seconds) unless it is newer than its sources
    and was built for the installed torch. Returns its path, or None without torch or g++."""
    torch_spec = importlib.util.find_spec("torch")
    if torch_spec is None or shutil.which("g++") is None:
        print(f"{os.path.basename(EXT)} is not built: {'g++' if torch_spec else 'torch'} is missing", file=sys.stderr)
        return None
    torch_dir = list(torch_spec.submodule_search_locations)[0]
    stamp = f"{torch_dir} {os.path.getmtime(os.path.join(torch_dir, 'version.py'))} {sys.version}\n"
    if not force and os.path.exists(EXT) and all(os.path.getmtime(x) <= os.path.getmtime(EXT) for x in EXT_SOURCES):
        with open(EXT, "rb") as f:
            f.seek(-min(os.path.getsize(EXT), len(stamp)), os.SEEK_END)
            if f.read() == stamp.encode():
                return EXT
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    abi = subprocess.run([sys.executable, "-c", "import torch; print(int(torch.compiled_with_cxx11_abi()))"], check=True,
                         capture_output=True, text=True).stdout.strip()
    with _written(EXT) as tmp:
        subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
                        "-I", INCLUDE, "-I", os.path.join(torch_dir, "include"),
                        "-I", os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
                        "-I", os.path.join(cuda, "include"), "-I", sysconfig.get_paths()["include"],
                        EXT_SOURCES[0], "-o", tmp, "-L", os.path.join(torch_dir, "lib"),
                        "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"], check=True)
        with open(tmp, "ab") as f:  # what it was built for, after the last byte that the loader reads
            f.write(stamp.encode())
    return EXT


def _sources():
    return sorted(
        [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))]
        + [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    )


def up_to_date(out=OUT):
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(s) <= t for s in _sources())


def nvcc():
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libgqa_sm100.so")
    return path


def build(force=False, verbose=False, debug=False):
    """Compiles the library (or, with debug, its checked variant) and the binding unless they
    are newer than every source. Returns the library's path."""
    out = OUT_DEBUG if debug else OUT
    if force or not up_to_date(out):
        with _written(out) as tmp:
            cmd = [nvcc(), *NVCC_FLAGS, *(["-DGQA_DEBUG_CHECKS"] if debug else []), "-I", INCLUDE, "-o", tmp,
                   os.path.join(CSRC, "gqa_sm100.cu")]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True)
    build_ext(force)
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    ap.add_argument("--debug", action="store_true", help="build libgqa_sm100_debug.so (in-kernel checks)")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose, debug=a.debug))
    sys.exit(0)
