"""Build libnomas_kv.so (C ABI + sm_100a kernels) and _block_binding.so (the
Python extension of nomas_kv/block.py, compiled against torch) in-tree.

    python hy-nomas-rs_b200/build.py          # incremental
    python hy-nomas-rs_b200/build.py --clean  # from scratch

Objects go to hy-nomas-rs_b200/_build/, the libraries to
hy-nomas-rs_b200/nomas_kv/ (both git-ignored; the .so travels
with the source tree to the GPU host).  nvcc cross-compiles for sm_100a, so
this runs on a machine without a GPU.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "nomas_kv", "libnomas_kv.so")
BINDING = os.path.join(PKG, "nomas_kv", "_block_binding.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

SOURCES = ["kernels_commit.cu", "kernels_gather.cu", "kernels_qvg.cu", "kernels_qvg_fit.cu", "kernels_project.cu",
           "kernels_attn.cu", "kernels_packed.cu", "kernels_rotary.cu", "kernels_norm.cu",
           "bank.cpp", "abi.cpp", "abi_block.cpp",
           "noalloc.cu"]
HEADERS = ["nkv_kernels.h", "nkv_device.cuh", "nkv_quant.cuh", "nkv_tcgen05.cuh", "nkv_policy.h", "nkv_packed.h",
           "bank.h"]

# -fmad=false / -ffp-contract=off: the reference rounds every multiply and
# add separately; the kernels ask for fused operations explicitly where the
# result is provably identical.
COMMON = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-fmad=false",
    "-Xcompiler", "-fPIC,-ffp-contract=off,-fno-fast-math,-Wall,-Wno-unused-function",
    "-I", os.path.join(ROOT, "include"), "-I", CSRC,
]


def _newer(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src: str) -> str:
    path = os.path.join(CSRC, src)
    obj = os.path.join(BUILD, src + ".o")
    deps = [path] + [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(ROOT, "include", "nomas_kv.h")]
    if _newer(obj, deps):
        cmd = [NVCC, *COMMON, "-c", path, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def _binding() -> None:
    """_block_binding.so holds torch's and Python's internals as they were when it
    was compiled: another version of either, or other flags, compile it anew."""
    import importlib.metadata
    import importlib.util
    import json
    import sysconfig

    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.origin:  # (a folder of that name has no origin)
        # without torch nothing can call the block operators of nomas_kv
        print("no torch: _block_binding.so not built", file=sys.stderr)
        return
    base = os.path.dirname(spec.origin)
    src, header = os.path.join(CSRC, "block_binding.cpp"), os.path.join(ROOT, "include", "nomas_kv.h")
    inc = [os.path.join(ROOT, "include"), os.path.join(base, "include"), sysconfig.get_paths()["include"],
           os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")]
    cmd = [os.environ.get("CXX", "g++"), "-shared", "-fPIC", "-O2", "-std=c++17", "-Wall", *(f"-isystem{i}" for i in inc),
           src, "-o", BINDING, f"-L{os.path.join(base, 'lib')}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_cuda",
           "-lc10"]
    stamp = os.path.join(BUILD, "block_binding.json")
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:  # a source tree: its version file says when it was built
        version = os.path.getmtime(os.path.join(base, "version.py"))
    made_for = json.dumps([version, sys.version, cmd]).replace(ROOT, "")
    try:
        with open(stamp) as f:
            current = f.read() == made_for
    except OSError:
        current = False
    if current and not _newer(BINDING, [src, header]):
        return
    if not current and os.path.exists(BINDING):
        os.remove(BINDING)  # of another torch: not to be loaded, even if the compiler fails now
    try:
        import torch
    except ImportError as e:
        raise RuntimeError(f"_block_binding.so is compiled against torch: {e}") from e

    cmd.insert(1, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}")
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"{e}: _block_binding.so needs a C++ compiler (CXX, default g++)") from e
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for block_binding.cpp:\n{r.stdout}\n{r.stderr}")
    with open(stamp, "w") as f:
        f.write(made_for)


def build(clean: bool = False, verbose: bool = False) -> str:
    if clean:
        shutil.rmtree(BUILD, ignore_errors=True)
        for made in (LIB, BINDING):
            if os.path.exists(made):
                os.remove(made)
    os.makedirs(BUILD, exist_ok=True)
    with ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as ex:
        binding = ex.submit(_binding)
        objs = list(ex.map(_compile, SOURCES))
    if _newer(LIB, objs):
        cmd = [NVCC, "-shared", "-cudart", "static", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB, *objs,
               "-lpthread", "-ldl", "-lrt"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(LIB)
    # last: the C library needs nvcc alone, and is there whether or not torch's
    # headers, Python's and a C++ compiler are
    binding.result()
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--clean", action="store_true")
    a = ap.parse_args()
    try:
        build(clean=a.clean, verbose=True)
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
