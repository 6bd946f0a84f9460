"""Build the MI355X library in-tree.

Outputs, next to this file (git-ignored, used in place):
  fa_kernels.hsaco  gfx950 code object with the attention kernels (hipcc --genco)
  fa_score_*.hsaco, fa_cache_*.hsaco (f32, bf16, f16), fa_rotary.hsaco
                    code objects of attention with modified scores, of the
                    key / value cache and of rotary positions
  libfa_hip.so      C ABI of include/fa_hip.h over the HIP runtime

All are written aside and moved into place together once every one of them has
compiled, so that a build that fails leaves the last one whole.  The operators'
code objects and the library carry a stamp of the parameter blocks that they
share, and the library loads no code object of another stamp.

Run as ``python flash-attention-cpu_amd/build.py`` or via
``__graft_entry__.build()``.  Needs only hipcc / amdclang++ from /opt/rocm;
cross-compiles for gfx950 without a GPU.
"""
from __future__ import annotations

import hashlib
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

# code objects of the operators: name -> (source, defines)
TYPES = {"f32": ("-DOPS_T=float", "-DOPS_NAME=f32"), "bf16": ("-DOPS_T=__bf16", "-DOPS_NAME=bf16", "-DOPS_16BIT"),
         "f16": ("-DOPS_T=_Float16", "-DOPS_NAME=f16", "-DOPS_16BIT")}
OBJECTS = {"fa_kernels": ("fa_kernels", ()), "fa_rotary": ("fa_rotary", ()),
           **{f"{src}_{t}": (src, flags) for src in ("fa_score", "fa_cache") for t, flags in TYPES.items()}}
LIB = os.path.join(HERE, "libfa_hip.so")
BUILD = os.path.join(HERE, "_build")   # intermediate objects, and outputs until all are there (git-ignored)

# -packed-fp32-ops: keep the compiler from emitting v_pk_{add,mul,fma}_f32.
HIP_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _run(cmd: list[str]) -> None:
    print("+", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def stamp() -> str:
    """Of the parameter blocks and the geometry that host and kernels of the operators share."""
    with open(os.path.join(CSRC, "fa_ops_params.h"), "rb") as f:
        return hashlib.sha256(f.read()).hexdigest()[:16]


def _aside(path: str) -> str:
    return os.path.join(BUILD, os.path.basename(path))


def build_object(name: str) -> str:
    src, flags = OBJECTS[name]
    out = os.path.join(HERE, name + ".hsaco")
    _run([os.path.join(ROCM, "bin", "hipcc"), *HIP_FLAGS, *flags, f"-DOPS_STAMP={stamp()}", "--genco",
          os.path.join(CSRC, src + ".hip"), "-o", _aside(out)])
    return out


def build_kernels() -> list[str]:
    """Every code object, compiled at the same time."""
    with ThreadPoolExecutor(max_workers=len(OBJECTS)) as pool:
        return list(pool.map(build_object, OBJECTS))


def build_host() -> list[str]:
    """libfa_hip.so: fa_host.cpp (host-only C++) plus fa_scratch.hip, whose
    object carries the device-global scratch array of the allocation-free
    entry point in an embedded gfx950 code object."""
    scratch_obj = os.path.join(BUILD, "fa_scratch.o")
    _run([os.path.join(ROCM, "bin", "hipcc"), *HIP_FLAGS, "-fPIC", "-Wall", "-Wextra", "-c",
          os.path.join(CSRC, "fa_scratch.hip"), "-o", scratch_obj])
    _run([os.path.join(ROCM, "llvm", "bin", "clang++"), "-D__HIP_PLATFORM_AMD__", f"-DOPS_STAMP={stamp()}",
          "-I", os.path.join(ROCM, "include"), "-fPIC", "-shared", "-O2", "-std=c++17",
          "-Wall", "-Wextra", os.path.join(CSRC, "fa_host.cpp"), scratch_obj,
          "-L", os.path.join(ROCM, "lib"), "-lamdhip64", "-Wl,-rpath," + os.path.join(ROCM, "lib"),
          "-o", _aside(LIB)])
    return [LIB]


def build(parts=(build_kernels, build_host)) -> None:
    os.makedirs(BUILD, exist_ok=True)
    outputs = [path for part in parts for path in part()]
    for path in outputs:
        os.replace(_aside(path), path)


if __name__ == "__main__":
    build()
    sys.exit(0)
