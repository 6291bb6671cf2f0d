"""Build the native libraries in-tree: ``stockfish_trainer_b200/libnnue_ft.so``
(the feature transformer) and ``libnnue_ls.so`` (the layer stacks).

    python -m stockfish_trainer_b200.build [--force] [--verbose]

For libnnue_ft.so one nvcc invocation compiles the CUDA kernels for sm_100a (nnue_ft.cu) and the
host-side position / feature-index code (features.cpp) into a single shared
library with a plain C ABI (include/nnue_ft.h).  ``-fmad=false`` keeps every
fp32 operation a separately rounded IEEE op, which the bit-exact parity with
the reference relies on.  libnnue_ls.so (csrc/layer_stacks/, include/nnue_ls.h)
is compiled without it: its sums are not tied to a reference order.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
import tempfile

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_NAME = "libnnue_ft.so"
LIB_PATH = os.path.join(PKG, LIB_NAME)

SOURCES = ["nnue_ft.cu", "features.cpp"]
DEPS = SOURCES + ["common.cuh", "ft_forward.cuh", "ft_backward.cuh", "ft_quant.cuh", "ft_epilogue.cuh",
                  "ft_optim.cuh", "ft_encode.cuh", "ft_exchange.cuh", "feature_tables.h", "feature_encode.h"]

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put CUDA's bin directory on PATH)")


LS_CSRC = os.path.join(CSRC, "layer_stacks")
LS_LIB_PATH = os.path.join(PKG, "libnnue_ls.so")


def _stale(lib: str, deps: list[str]) -> bool:
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    return any(os.path.getmtime(d) > t for d in deps)


def _nvcc(args: list[str], verbose: bool) -> None:
    cmd = [nvcc(), *ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC,-O3,-pthread", "-I", INCLUDE, *args]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)
    if verbose:
        sys.stderr.write(res.stderr)


def build(force: bool = False, verbose: bool = False) -> str:
    deps = [os.path.join(CSRC, d) for d in DEPS] + [os.path.join(INCLUDE, "nnue_ft.h")]
    if not force and not _stale(LIB_PATH, deps):
        return LIB_PATH
    tmp = LIB_PATH + ".tmp"
    _nvcc(["-fmad=false", "-shared", *(os.path.join(CSRC, s) for s in SOURCES), "-o", tmp, "-lpthread"], verbose)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def build_layer_stacks(force: bool = False, verbose: bool = False) -> str:
    deps = [os.path.join(LS_CSRC, d) for d in sorted(os.listdir(LS_CSRC)) if d.endswith((".cu", ".cuh"))]
    if not force and not _stale(LS_LIB_PATH, deps + [os.path.join(INCLUDE, "nnue_ls.h")]):
        return LS_LIB_PATH
    sources = sorted(d for d in os.listdir(LS_CSRC) if d.endswith(".cu"))
    tmp = LS_LIB_PATH + ".tmp"
    with tempfile.TemporaryDirectory() as objects:  # one nvcc per source file, side by side
        outs = [os.path.join(objects, s + ".o") for s in sources]
        with concurrent.futures.ThreadPoolExecutor(len(sources)) as pool:
            list(pool.map(lambda so: _nvcc(["-c", os.path.join(LS_CSRC, so[0]), "-o", so[1]], verbose),
                          zip(sources, outs)))
        _nvcc(["-shared", *outs, "-o", tmp, "-lpthread"], verbose)
    os.replace(tmp, LS_LIB_PATH)
    return LS_LIB_PATH


if __name__ == "__main__":
    for fn in (build, build_layer_stacks):
        print(fn(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
