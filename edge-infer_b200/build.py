"""Builds the sm_100a shared library in-tree with nvcc (cross-compiles without a GPU).

    python edge-infer_b200/build.py            # incremental
    python edge-infer_b200/build.py --force

Output: edge-infer_b200/libedge_infer_b200.so and _calls with the interpreter's suffix, the Python calls that take torch
tensors apart natively (both git-ignored; they travel with the tree). Where Python's headers are not installed only the library
is built: hosts that link it need no more, and the operators that go through the native calls say what is missing.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OBJ = HERE / "build"
LIB = HERE / "libedge_infer_b200.so"
CALLS = HERE / ("_calls" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))  # another interpreter's is not loaded
SOURCES = ["abi_ops.cu", "smallm_gemm.cu", "prompt_gemm.cu", "elementwise.cu", "attention.cu", "sampling.cu", "runtime.cu",
           "layered.cu", "layered_kernels.cu", "lightning.cu", "sized_attention.cu",
           "parallel_block.cu", "outer_state.cu", "latent_attention.cu", "delta_prompt.cu",
           "context_ops.cu", "qk_rope.cu", "step_attention.cu", "span_attention.cu", "evict.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
]


def _newest_dependency() -> float:
    paths = list(CSRC.glob("*")) + [HERE.parent / "include" / "edge_infer_b200.h", Path(__file__)]
    return max(p.stat().st_mtime for p in paths)


def _python_headers() -> Path | None:
    include = Path(sysconfig.get_paths()["include"])
    return include if (include / "Python.h").exists() else None


def _build_calls() -> None:
    include = _python_headers()
    if include is None:
        print(f"{sysconfig.get_paths()['include']} has no Python.h: {CALLS.name} is not built", file=sys.stderr)
        return
    calls = [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared", "-I" + str(include),
             str(CSRC / "python_calls.cpp"), "-o", str(CALLS), "-L" + str(HERE), "-ledge_infer_b200", "-Wl,-rpath,$ORIGIN"]
    result = subprocess.run(calls, capture_output=True, text=True)
    if result.returncode:
        raise RuntimeError(f"compilation of the Python calls failed:\n{result.stdout}\n{result.stderr}")
    if CALLS.name != "_calls.so":
        (HERE / "_calls.so").unlink(missing_ok=True)  # of any interpreter: an earlier build's name


def _compile(source: str, verbose: bool) -> None:
    out = OBJ / (source + ".o")
    cmd = [NVCC, *FLAGS, "-c", str(CSRC / source), "-o", str(out)]
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
    result = subprocess.run(cmd, capture_output=True, text=True)
    if verbose and result.stderr:
        (OBJ / (source + ".ptxas.txt")).write_text(result.stderr)
    if result.returncode:
        raise RuntimeError(f"nvcc failed for {source}:\n{result.stdout}\n{result.stderr}")


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles every CUDA source for sm_100a and links the shared library."""
    newest = _newest_dependency()
    wanted = (LIB, CALLS) if _python_headers() else (LIB,)
    if not force and all(p.exists() and p.stat().st_mtime >= newest for p in wanted):
        return LIB
    OBJ.mkdir(exist_ok=True)
    stale = [s for s in SOURCES
             if force or not (OBJ / (s + ".o")).exists() or (OBJ / (s + ".o")).stat().st_mtime < _newest_dependency()]
    with ThreadPoolExecutor(max_workers=min(8, len(stale) or 1)) as pool:
        list(pool.map(lambda s: _compile(s, verbose), stale))
    objects = [str(OBJ / (s + ".o")) for s in SOURCES]
    link = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", str(LIB), *objects,
            "-lcudart"]
    result = subprocess.run(link, capture_output=True, text=True)
    if result.returncode:
        raise RuntimeError(f"link failed:\n{result.stdout}\n{result.stderr}")
    _build_calls()
    return LIB


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
