"""Builds libtabicl_attn.so (the C-ABI HIP library) for gfx950 with hipcc, and tabicl_mi355_direct.so (a Python module that
makes the paged cache's calls of it, csrc/direct.cpp; host code alone) with g++, in-tree. The library needs neither torch nor
Python; where these, their headers or g++ are missing, a warning says so and the module is left out (the wrappers call the library
by ctypes then).

Usage: python build_lib.py [-v]. Objects go to _build/ next to this file; the library is written
next to this file, where tabicl_mi355_native.py loads it from.
"""
from __future__ import annotations

import concurrent.futures
import os
import subprocess
import sys
import warnings
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
BUILD = HERE / "_build"
LIB = HERE / "libtabicl_attn.so"
DIRECT = HERE / "tabicl_mi355_direct.so"
CXX = os.environ.get("CXX", "g++")
ARCH = "gfx950"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 in any kernel of this library.
# -amdgpu-mfma-vgpr-form: MFMA results in arch VGPRs; the default AGPR form makes the compiler copy
#  every accumulator between AGPRs and VGPRs around the softmax (measured: ~128 copies per tile).
FLAGS = ["-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}", "-Xclang", "-target-feature",
         "-Xclang", "-packed-fp32-ops", "-mllvm", "-amdgpu-mfma-vgpr-form", "-Wall", "-Wno-unused-function",
         "-Wno-unused-command-line-argument"]
SOURCES = ["abi.hip", "icl_fwd.hip", "icl_bwd.hip", "smallhead_fwd.hip", "smallhead_split.hip", "smallhead_rows.hip", "smallhead_stream.hip", "smallhead_bwd.hip", "keymask.hip",
           "layernorm.hip", "layer.hip", "icl_layer.hip", "paged.hip", "paged_q8.hip", "paged_sparse.hip", "paged_books.hip"]


def _compile(src: Path, obj: Path, verbose: bool) -> None:
    cmd = [HIPCC, *FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{res.stderr}")
    if verbose and res.stderr.strip():
        print(res.stderr, flush=True)


def _direct(verbose: bool) -> Path:
    import sysconfig

    import torch
    torch_dir = Path(torch.__file__).resolve().parent
    tmp = DIRECT.with_suffix(".so.tmp")
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{sysconfig.get_paths()['include']}", f"-isystem{torch_dir / 'include'}",
           f"-isystem{torch_dir / 'include' / 'torch' / 'csrc' / 'api' / 'include'}", str(CSRC / "direct.cpp"), "-o", str(tmp),
           f"-L{torch_dir / 'lib'}", "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for direct.cpp:\n{res.stderr}")
    return tmp


def build(verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    objs = [BUILD / (Path(s).stem + ".o") for s in SOURCES]
    with concurrent.futures.ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as ex:
        futs = [ex.submit(_compile, CSRC / s, o, verbose) for s, o in zip(SOURCES, objs)]
        direct = ex.submit(_direct, verbose)
        for f in futs:
            f.result()
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, LIB)
    try:
        os.replace(direct.result(), DIRECT)
    except (ImportError, OSError, RuntimeError) as e:
        DIRECT.unlink(missing_ok=True)  # one of another library would call it by other signatures
        warnings.warn(f"{DIRECT.name} was not built, the paged cache's calls go by ctypes: {e}", RuntimeWarning)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
