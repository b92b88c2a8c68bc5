"""Compile libmoe_gfx950.so (HIP, gfx950) in-tree, and attn_binding.so, the Python
binding of a few of its entry points.

Each csrc/*.hip file is compiled to an object under _build/ (in parallel), then
linked into gpt-oss-tvm_amd/libmoe_gfx950.so next to this file.  hipcc
cross-compiles for gfx950 without a GPU.  csrc/attn_binding.cpp is host code over torch's
C++ API, compiled beside them and linked against that library.

    python gpt-oss-tvm_amd/build_native.py
"""
from __future__ import annotations

import concurrent.futures
import glob
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libmoe_gfx950.so")
BINDING = os.path.join(HERE, "attn_binding.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

# Packed fp32 ops stay off: hipcc would otherwise form v_pk_{add,mul,fma}_f32
# from ordinary float code.
FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden",
    "-Wall", "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{INCLUDE}",
]


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.basename(src).replace(".hip", ".o"))
    cmd = [HIPCC, *FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def _run(cmd: list, what: str) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{r.stdout}\n{r.stderr}")


def _torch_lib() -> str:
    import torch
    return os.path.join(os.path.dirname(torch.__file__), "lib")


def _compile_binding() -> str:
    import torch
    include = os.path.join(os.path.dirname(torch.__file__), "include")
    obj = os.path.join(BUILD, "attn_binding.o")
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Wall",
          "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-DTORCH_API_INCLUDE_EXTENSION_H",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
          "-isystem", include, "-isystem", os.path.join(include, "torch", "csrc", "api", "include"),
          "-isystem", "/opt/rocm/include", "-isystem", sysconfig.get_paths()["include"],
          "-c", os.path.join(CSRC, "attn_binding.cpp"), "-o", obj], "attn_binding.cpp")
    return obj


def build(verbose: bool = True) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        binding = ex.submit(_compile_binding)
        objs = list(ex.map(_compile, srcs))
    tmp = LIB + ".tmp"
    _run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", tmp], "link")
    os.replace(tmp, LIB)
    tmp = BINDING + ".tmp"
    lib = _torch_lib()
    _run(["g++", "-shared", "-fPIC", binding.result(), "-o", tmp, f"-L{lib}", "-ltorch_python",
          "-ltorch_cpu", "-lc10", "-lc10_hip", f"-L{HERE}", "-l:" + os.path.basename(LIB),
          "-Wl,-rpath,$ORIGIN"], "link of attn_binding")
    os.replace(tmp, BINDING)
    if verbose:
        print(f"built {LIB} from {len(srcs)} sources, and {BINDING}", flush=True)
    return LIB


if __name__ == "__main__":
    build()
    sys.exit(0)
