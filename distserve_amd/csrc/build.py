"""Builds the two shared libraries of the package, in-tree, for gfx950.

``libkvmove.so``        hand-written HIP kernels + the C ABI (``include/kvmove.h``); no torch.  Migration and
                        swap are ``kvmove.hip``, the cache operators ``kvcache*.hip`` and ``kvcache_plan.cpp``.
``libkvmove_torch.so``  torch op shim registering ``block_migration_ops`` / ``swapping_ops`` (``kvmove_torch.cpp``)
                        and ``kvcache_ops`` (``kvcache_torch.cpp``).
``tests/lib_explore/libkvmove.so``  the HIP library again with ``-DKVM_EXPLORE``: every kernel flavour and the
                        knobs that select them, for sweeps and for the tests that show every flavour copies the
                        same bytes.  Never loaded by the package.
``libkvmove_torch_alt.so``  the same ops as ``kvmove_block_migration_ops`` / ``kvmove_swapping_ops`` / ``kvmove_kvcache_ops``,
                        for a process that keeps another registration of DistServe's names.

Run as ``python distserve_amd/csrc/build.py`` (a plain script on purpose: it must work
when the libraries are missing or stale, so it does not import the package, which loads
them).  hipcc cross-compiles without a GPU.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

CSRC_DIR = os.path.dirname(os.path.abspath(__file__))
PKG_DIR = os.path.dirname(CSRC_DIR)
REPO_DIR = os.path.dirname(PKG_DIR)
LIB_DIR = os.path.join(PKG_DIR, "lib")
OBJ_DIR = os.path.join(CSRC_DIR, "build")
INCLUDE_DIR = os.path.join(REPO_DIR, "include")

KVMOVE_LIB = os.path.join(LIB_DIR, "libkvmove.so")
TORCH_LIB = os.path.join(LIB_DIR, "libkvmove_torch.so")
TORCH_ALT_LIB = os.path.join(LIB_DIR, "libkvmove_torch_alt.so")
EXPLORE_LIB = os.path.join(REPO_DIR, "tests", "lib_explore", "libkvmove.so")
ALT_NAMESPACES = ("kvmove_block_migration_ops", "kvmove_swapping_ops", "kvmove_kvcache_ops")

GPU_ARCH = "gfx950"
ROCM_HOME = os.environ.get("ROCM_PATH", "/opt/rocm")


def _run(cmd):
    print("+", " ".join(cmd), flush=True)
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    # the host pass of hipcc does not know the packed-fp32 target feature and says so
    out = "\n".join(l for l in res.stdout.splitlines() if "packed-fp32-ops" not in l)
    if out.strip():
        print(out, flush=True)
    if res.returncode != 0:
        raise RuntimeError(f"build step failed with exit code {res.returncode}: {' '.join(cmd)}")


def _hipcc() -> str:
    return shutil.which("hipcc") or os.path.join(ROCM_HOME, "bin", "hipcc")


def _object(source: str, name: str, *flags: str) -> str:
    out = os.path.join(OBJ_DIR, name)
    os.makedirs(OBJ_DIR, exist_ok=True)
    _run([
        _hipcc(), f"--offload-arch={GPU_ARCH}", "-O3", "-std=c++17", "-fPIC", "-c",
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-Wall", "-Wextra", f"-I{INCLUDE_DIR}", *flags, os.path.join(CSRC_DIR, source), "-o", out,
    ])
    return out


def _objects(specs):
    """Compiles the translation units side by side."""
    with ThreadPoolExecutor(max_workers=4) as pool:
        return list(pool.map(lambda spec: _object(*spec), specs))


CACHE_UNITS = [("kvcache.hip", "kvcache.o"), ("kvcache_tiles.hip", "kvcache_tiles.o"), ("kvcache_plan.cpp", "kvcache_plan.o")]


def build_kvmove(explore: bool = False, cache_objects=None) -> str:
    """libkvmove.so from its translation units; the exploration build shares the cache operators' objects."""
    out = EXPLORE_LIB if explore else KVMOVE_LIB
    os.makedirs(os.path.dirname(out), exist_ok=True)
    move = ("kvmove.hip", "kvmove_explore.o", "-DKVM_EXPLORE") if explore else ("kvmove.hip", "kvmove.o")
    objects = _objects([move] + ([] if cache_objects else CACHE_UNITS))
    _run([_hipcc(), f"--offload-arch={GPU_ARCH}", "-shared", "-fPIC", *objects, *(cache_objects or []), "-o", out])
    return out


def build_torch_shim(alt: bool = False) -> str:
    import torch
    from torch.utils import cpp_extension

    if not os.path.exists(KVMOVE_LIB):
        build_kvmove()
    torch_lib_dir = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{INCLUDE_DIR}", f"-I{os.path.join(ROCM_HOME, 'include')}"]
    cmd += [f"-I{p}" for p in cpp_extension.include_paths()]
    out = TORCH_LIB
    if alt:
        out = TORCH_ALT_LIB
        cmd += [f"-DKVM_MIGRATION_NS={ALT_NAMESPACES[0]}", f"-DKVM_SWAP_NS={ALT_NAMESPACES[1]}",
                f"-DKVM_CACHE_NS={ALT_NAMESPACES[2]}"]
    cmd += [os.path.join(CSRC_DIR, "kvmove_torch.cpp"), os.path.join(CSRC_DIR, "kvcache_torch.cpp"), "-o", out,
            f"-L{LIB_DIR}", "-lkvmove", "-Wl,-rpath,$ORIGIN",
            f"-L{torch_lib_dir}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch", "-Wl,--no-as-needed"]
    _run(cmd)
    return out


def build_all() -> None:
    cache_objects = _objects(CACHE_UNITS)
    build_kvmove(cache_objects=cache_objects)
    build_kvmove(explore=True, cache_objects=cache_objects)
    with ThreadPoolExecutor(max_workers=2) as pool:
        list(pool.map(lambda alt: build_torch_shim(alt=alt), (False, True)))


if __name__ == "__main__":
    build_all()
    print("built:", KVMOVE_LIB, TORCH_LIB, TORCH_ALT_LIB, EXPLORE_LIB)
    sys.exit(0)
