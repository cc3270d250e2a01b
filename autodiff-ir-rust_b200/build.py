"""Builds libadb200.so in-tree (csrc/ -> autodiff-ir-rust_b200/libadb200.so) with nvcc for sm_100a.

    python autodiff-ir-rust_b200/build.py [--force] [--verbose]

nvcc cross-compiles without a GPU; the result travels with the source tree.  NVRTC is linked
dynamically from the CUDA toolkit (the generated kernels are compiled at first use), cudart is linked
statically, libcuda and libnccl are not linked at all (entry points are fetched at run time).
"""
from __future__ import annotations

import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libadb200.so")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
SOURCES = ["adb_runtime.cu", "adb_gemm.cu", "adb_noalloc.cu", "adb_norm.cu", "adb_rotary.cu", "adb_attention.cu", "adb_attention_tc.cu", "adb_attention_decode.cu",
           "adb_lower.cpp", "adb_codegen.cpp", "adb_shard.cpp"]


def needs_build() -> bool:
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    for root in (CSRC, os.path.join(os.path.dirname(HERE), "include")):
        for f in os.listdir(root):
            if os.path.getmtime(os.path.join(root, f)) > t:
                return True
    return False


def check_register_shares(ptxas: str, source: str) -> None:
    """The key-gradient kernels hand registers from some of their warps to the others (setmaxnreg), out of what the block is
    launched with: a variant that the compiler gave fewer than KEY_REGS would wait for them for good.  `ptxas` is what
    `-Xptxas=-v` printed, `source` the file that says KEY_REGS."""
    need = int(re.search(r"\bKEY_REGS = (\d+)", source).group(1))
    used = [int(n) for n in re.findall(r"Compiling entry function '\S*adb_attention_tc_dkv\S*'.*?Used (\d+) registers", ptxas, re.S)]
    if not used:
        raise RuntimeError("the compiler's report names no key-gradient kernel")
    if min(used) < need:
        raise RuntimeError(f"a key-gradient kernel has {min(used)} registers a thread, its warps share out {need}")


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return OUT
    cmd = [
        os.path.join(CUDA, "bin", "nvcc"), "-O3", "-std=c++17",
        "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
        "-Xptxas=-v", "-Xcompiler", "-fPIC,-Wall,-Wextra,-Wno-unused-parameter", "-shared",
        "-o", OUT,
    ] + [os.path.join(CSRC, s) for s in SOURCES] + [
        "-lnvrtc", "-ldl", "-Xlinker", f"-rpath={CUDA}/lib64",
    ]
    if verbose:
        print(" ".join(cmd))
    run = subprocess.run(cmd, stderr=subprocess.PIPE, text=True)
    sys.stderr.writelines(l for l in run.stderr.splitlines(True) if verbose or run.returncode or "warning" in l)
    run.check_returncode()
    with open(os.path.join(CSRC, "adb_attention_tc.cu")) as f:
        try:
            check_register_shares(run.stderr, f.read())
        except RuntimeError:
            os.remove(OUT)
            raise
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
