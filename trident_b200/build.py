"""Builds libtb200.so (the C-ABI kernel library) in-tree with nvcc for sm_100a.

Usage: python -m trident_b200.build [--force] [--verbose]
"""

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ_DIR = os.path.join(HERE, "build")
LIB_PATH = os.path.join(HERE, "libtb200.so")
# direct Python entry points (csrc/fastcall.c), of the interpreter that builds them
FASTCALL_PATH = os.path.join(HERE, "_fastcall" + sysconfig.get_config_var("EXT_SUFFIX"))

SOURCES = [
    "api.cu",
    "row_norm.cu",
    "residual_norm.cu",
    "softmax.cu",
    "reduce.cu",
    "gemm_simt.cu",
    "gemm_tc.cu",
    "attention_simt.cu",
    "attention_fwd_tc.cu",
    "attention_bwd_tc.cu",
    "local_attention.cu",
    "local_attention_simt.cu",
    "local_attention_fwd_tc.cu",
    "local_attention_bwd_tc.cu",
    "local_attention_few_tc.cu",
]

NVCC_FLAGS = [
    "-std=c++17",
    "-O3",
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
    "--expt-relaxed-constexpr",
    "-Xptxas",
    "-v",
]


def _nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _headers():
    out = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    out.append(os.path.join(HERE, "..", "include", "tb200.h"))
    return out


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _compile(src, force, verbose):
    obj = os.path.join(OBJ_DIR, src.replace(".cu", ".o"))
    path = os.path.join(CSRC, src)
    if not force and not _stale(obj, [path] + _headers()):
        return obj, ""
    cmd = [_nvcc(), *NVCC_FLAGS, "-c", path, "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{res.stdout}\n{res.stderr}")
    log = res.stderr
    with open(obj + ".ptxas.log", "w") as f:
        f.write(log)
    if verbose:
        sys.stderr.write(log)
    return obj, log


def build(force=False, verbose=False):
    """Compiles every .cu file and links libtb200.so; returns the library path."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(8, len(SOURCES))) as pool:
        results = list(pool.map(lambda s: _compile(s, force, verbose), SOURCES))
    objs = [r[0] for r in results]
    if force or _stale(LIB_PATH, objs):
        cmd = [_nvcc(), "-shared", "-o", LIB_PATH, *objs, "-lcudart", "-Xlinker", "-z,defs", "-Xlinker", "-soname,libtb200.so"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    _build_fastcall(force)
    return LIB_PATH


def _build_fastcall(force):
    """The CPython extension beside the library, linked against it. Where there is no C compiler or no Python headers
    the calls go through ctypes instead: the same kernels, 5 us more of host time a call."""
    source = os.path.join(CSRC, "fastcall.c")
    untagged = os.path.join(os.path.dirname(FASTCALL_PATH), "_fastcall.so")
    if os.path.exists(untagged):
        os.remove(untagged)  # (any interpreter would load it)
    if not force and not _stale(FASTCALL_PATH, [source, LIB_PATH, os.path.join(HERE, "..", "include", "tb200.h")]):
        return
    cmd = [
        os.environ.get("CC", "gcc"), "-std=c11", "-O2", "-Wall", "-shared", "-fPIC",
        "-I" + sysconfig.get_paths()["include"], source, "-o", FASTCALL_PATH,
        LIB_PATH, "-Wl,-rpath,$ORIGIN",
    ]
    try:
        res = subprocess.run(cmd, capture_output=True, text=True)
        failed = res.returncode != 0 and f"{res.stdout}\n{res.stderr}"
    except OSError as error:
        failed = str(error)
    if failed:
        if os.path.exists(FASTCALL_PATH):
            os.remove(FASTCALL_PATH)  # (out of date)
        print(f"the direct Python entry points are not built, calls go through ctypes:\n{failed}", file=sys.stderr)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
