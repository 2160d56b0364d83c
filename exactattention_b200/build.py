"""Builds libexactattn_cuda.so in-tree for sm_100a: python -m exactattention_b200.build

Each source compiles to its own object (in parallel, under _build/), then one link makes the
shared library. Objects are rebuilt when their source or any header changed."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
OUT = os.path.join(HERE, "libexactattn_cuda.so")
SOURCES = ["ea_simt.cu", "ea_tc.cu", "ea_decode.cu", "ea_api.cu", "ea_synth.cu", "ea_noalloc.cu", "ea_cache.cu",
           "ea_selftest.cu", "ea_nccl.cu", "ea_plan.cu", "ea_rope.cu", "ea_tree.cu",
           "ea_tree_tc.cu", "ea_logits.cu"]
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC"]
HEADERS = [os.path.join(HERE, "..", "include", f) for f in ("exactattn_cuda.h", "exactattn_serving.h")]


def _headers_mtime() -> float:
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))] + HEADERS
    return max(os.path.getmtime(p) for p in hs if os.path.exists(p))


def needs_build() -> bool:
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    return _headers_mtime() > t or any(os.path.getmtime(os.path.join(CSRC, f)) > t for f in SOURCES)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        build_synth_host()
        build_serving_native()
        return OUT
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    os.makedirs(OBJ, exist_ok=True)
    hdr = _headers_mtime()

    def compile_one(src: str) -> str:
        obj = os.path.join(OBJ, src.replace(".cu", ".o"))
        s = os.path.join(CSRC, src)
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(s), hdr):
            cmd = [nvcc, *FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-c", "-o", obj + ".tmp", src]
            subprocess.run(cmd, cwd=CSRC, check=True)
            os.replace(obj + ".tmp", obj)
        return obj

    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 4)) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    tmp = OUT + ".tmp"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC",
                    "-o", tmp, *objs], check=True)
    os.replace(tmp, OUT)
    build_synth_host(force)
    build_serving_native(force)
    return OUT


SYNTH_HOST = os.path.join(HERE, "libea_synth_host.so")


def build_synth_host(force: bool = False) -> str:
    """The host input generator (benchmarks and tests only), gcc with OpenMP."""
    src = os.path.join(CSRC, "ea_synth_host.c")
    if force or not os.path.exists(SYNTH_HOST) or os.path.getmtime(SYNTH_HOST) < os.path.getmtime(src):
        subprocess.run(["gcc", "-O3", "-fopenmp", "-fPIC", "-shared", "-o", SYNTH_HOST + ".tmp", src], check=True)
        os.replace(SYNTH_HOST + ".tmp", SYNTH_HOST)
    return SYNTH_HOST


SERVING_NATIVE = os.path.join(HERE, "_serving_native" + sysconfig.get_config_var("EXT_SUFFIX"))


def _serving_native_current(so: str) -> bool:
    """Whether the binding is newer than its sources and was built against the torch that is installed: its ABI is
    torch's C++ ABI, which changes from version to version. The version is in the module's `torch_version` string."""
    deps = [os.path.join(CSRC, "ea_serving_py.cpp"), HEADERS[1]]
    if not os.path.exists(so) or os.path.getmtime(so) < max(map(os.path.getmtime, deps)):
        return False
    import torch

    with open(so, "rb") as f:
        return f"built against torch {torch.__version__}\0".encode() in f.read()


def build_serving_native(force: bool = False) -> str:
    """The Python binding of the serving operators (csrc/ea_serving_py.cpp), g++ against torch's headers; it
    finds libexactattn_cuda.so beside itself. Without torch, which the rest of the package needs only for torch
    tensors, it is left out."""
    try:
        import torch
    except ImportError:
        print("no torch: the Python binding of the serving operators is not built", file=sys.stderr)
        return SERVING_NATIVE
    if force or not _serving_native_current(SERVING_NATIVE):
        from torch.utils import cpp_extension

        cuda = os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"))
        inc = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
        lib = cpp_extension.library_paths()
        subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f'-DEA_TORCH_VERSION="{torch.__version__}"',
                        *[f"-I{p}" for p in inc], "-o", SERVING_NATIVE + ".tmp", os.path.join(CSRC, "ea_serving_py.cpp"),
                        *[f"-L{p}" for p in lib], f"-L{HERE}", "-l:libexactattn_cuda.so", "-lc10", "-lc10_cuda",
                        "-ltorch_cpu",
                        "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"], check=True)
        os.replace(SERVING_NATIVE + ".tmp", SERVING_NATIVE)
    return SERVING_NATIVE


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
