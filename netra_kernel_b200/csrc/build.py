"""Builds libnetra_sm100.so (kernels + C ABI) for sm_100a with nvcc, and _netra_torch.so (torch side of the dense and
balance-loss entry points, host code only) with g++, in-tree.

Usage: python -m netra_kernel_b200.csrc.build [--verbose]
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
LIB = HERE / "libnetra_sm100.so"
CUBIN = HERE / "netra_moe_sm100a.cubin"
BINDING = HERE / "_netra_torch.so"
BINDING_DEPENDS = ["torch_binding.cpp", "../../include/netra_moe.h"]
SOURCES = ["api.cu", "engine.cpp"]
DEPENDS = ["api.cu", "engine.cpp", "kernels_cubin.cu", "common.cuh", "route_kernels.cu", "bridge_kernels.cu",
           "umma_kernels.cu", "umma_tokmajor.cu", "router_umma.cu", "ep_kernels.cu", "mxfp4_kernels.cu", "ep_p2p.cu", "static_scratch_sort.cu", "prefill_m768_bridge.cu",
           "dense_fp8.cu", "dense_pair.cu", "dense_few.cu", "balance.cu", "../../include/netra_moe.h", "../../include/netra_engine.h"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-ccbin", "g++"]
NVCC_FLAGS = [*ARCH_FLAGS, "--shared", "-Xcompiler", "-fPIC", "-Xptxas", "-v"]


def stale() -> bool:
    if not LIB.exists() or not CUBIN.exists() or not BINDING.exists():
        return True
    built = min(LIB.stat().st_mtime, CUBIN.stat().st_mtime)
    return any((HERE / d).stat().st_mtime > built for d in DEPENDS) or any((HERE / d).stat().st_mtime > BINDING.stat().st_mtime for d in BINDING_DEPENDS)


def binding_command() -> list[str]:
    """g++ line of the torch binding; it finds libnetra_sm100.so beside itself and torch's libraries in the process."""
    from torch.utils import cpp_extension
    includes = [*cpp_extension.include_paths(), "/usr/local/cuda/include", sysconfig.get_paths()["include"]]
    libs = cpp_extension.library_paths()
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", *[f"-I{i}" for i in includes], "-o", str(BINDING), str(HERE / "torch_binding.cpp"), *[f"-L{path}" for path in libs], f"-L{HERE}",
            "-L/usr/local/cuda/lib64", "-l:libnetra_sm100.so", "-lcudart", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not stale():
        return LIB
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    cmd = [nvcc, *NVCC_FLAGS, "-o", str(LIB), *[str(HERE / s) for s in SOURCES], "-lcudart"]
    proc = subprocess.run(cmd, capture_output=True, text=True, cwd=HERE)
    log = proc.stdout + proc.stderr
    (HERE / "build.log").write_text(log)
    if verbose or proc.returncode != 0:
        print(log)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed building libnetra_sm100.so (see csrc/build.log)")
    # the same kernels as a stand-alone code object for the engine runtime (cuModuleLoadData)
    cmd = [nvcc, *ARCH_FLAGS, "-cubin", "-o", str(CUBIN), str(HERE / "kernels_cubin.cu")]
    proc = subprocess.run(cmd, capture_output=True, text=True, cwd=HERE)
    (HERE / "build_cubin.log").write_text(proc.stdout + proc.stderr)
    if proc.returncode != 0:
        if verbose:
            print(proc.stdout + proc.stderr)
        raise RuntimeError("nvcc failed building netra_moe_sm100a.cubin (see csrc/build_cubin.log)")
    # host code against the C ABI: a change of the kernels does not touch it
    if not force and BINDING.exists() and BINDING.stat().st_mtime > max((HERE / d).stat().st_mtime for d in BINDING_DEPENDS):
        return LIB
    proc = subprocess.run(binding_command(), capture_output=True, text=True, cwd=HERE)
    (HERE / "build_binding.log").write_text(proc.stdout + proc.stderr)
    if proc.returncode != 0:
        if verbose:
            print(proc.stdout + proc.stderr)
        raise RuntimeError("g++ failed building _netra_torch.so (see csrc/build_binding.log)")
    return LIB


if __name__ == "__main__":
    build(force=True, verbose="--verbose" in sys.argv)
    print(LIB)
