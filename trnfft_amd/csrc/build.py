"""Build libtrnfft_amd.so (all HIP kernels + the C ABI) for gfx950 with hipcc, in-tree, and
libtfa_copy.so, the plain-copy kernels bench.py measures the achievable memory rate with; and, with the host compiler,
_tensor_table.so, which reads lists of tensors for the operators that take them, and _state_space.so, which makes the state space
operators' calls and their nodes of autograd's graph.

Usage: python -m trnfft_amd.csrc.build   (or trnfft_amd.csrc.build.build()).
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
LIB = os.path.join(PKG, "libtrnfft_amd.so")
COPY_LIB = os.path.join(PKG, "libtfa_copy.so")
COPY_SOURCE = "bench_copy.hip"
TABLE_LIB = os.path.join(PKG, "_tensor_table.so")
TABLE_SOURCE = "tensor_table.cpp"
SPACE_LIB = os.path.join(PKG, "_state_space.so")
SPACE_SOURCE = "state_space_calls.cpp"
SOURCES = [
    "plan.hip",
    "kernels_c2c.hip",
    "kernels_strided.hip",
    "kernels_bluestein.hip",
    "kernels_stft.hip",
    "kernels_stft_blue.hip",
    "kernels_gemm.hip",
    "kernels_fft2.hip",
    "kernels_real.hip",
    "kernels_istft.hip",
    "kernels_smooth_stft.hip",
    "kernels_smooth_istft.hip",
    "kernels_smooth_c2c.hip",
    "model_ops.hip",
    "kernels_attention.hip",
    "kernels_attention_f32.hip",
    "kernels_attention_bf16.hip",
    "kernels_attention_f16.hip",
    "kernels_norm.hip",
    "kernels_adamw.hip",
    "state_space_ops.hip",
    "kernels_conv.hip",
    "kernels_scan.hip",
    "kernels_scan_f32.hip",
    "kernels_scan_bf16.hip",
    "kernels_scan_f16.hip",
    "kernels_clip.hip",
]

CXX = os.environ.get("CXX", "g++")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
FLAGS = [
    "-O3",
    "--offload-arch=gfx950",
    "-std=c++17",
    "-fPIC",
    # no packed-fp32 (v_pk_*_f32) code generation: some of its forms gave wrong results now and then
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-function",
]


# per-source extra flags: the fused Bluestein kernels feed compile-time zeros (the zero-padded
# half of its forward input) into its first pass; ignoring the sign of zero lets the compiler drop
# the additions of those zeros (x + 0 -> x), which changes no result beyond the sign of a zero
EXTRA_FLAGS = {"kernels_bluestein.hip": ["-fno-signed-zeros"], "kernels_stft_blue.hip": ["-fno-signed-zeros"]}


def _compile(src: str, obj: str) -> None:
    cmd = [HIPCC, *FLAGS, *EXTRA_FLAGS.get(src, []), "-c", os.path.join(HERE, src), "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{res.stderr}")


def _link(objs: list[str], out: str) -> None:
    tmp = out + ".tmp"
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", tmp]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed for {os.path.basename(out)}:\n{res.stderr}")
    os.replace(tmp, out)


def _build_module(src: str, out: str) -> None:
    """A CPython module on torch's own headers (torch is loaded before it: its libraries need no search path)."""
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    tmp = out + ".tmp"
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"]
    for path in (*include_paths(), os.path.join(ROCM, "include"), sysconfig.get_path("include")):
        cmd += ["-isystem", path]
    cmd += [os.path.join(HERE, src), "-o", tmp, *(f"-L{p}" for p in library_paths()), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_hip"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{CXX} failed for {src}:\n{res.stderr}")
    os.replace(tmp, out)


def _build_table() -> None:
    _build_module(TABLE_SOURCE, TABLE_LIB)


def _build_state_space() -> None:
    _build_module(SPACE_SOURCE, SPACE_LIB)


def build(verbose: bool = False) -> str:
    """Compile every source and link the shared libraries; returns the main library's path."""
    if not shutil.which(HIPCC) and not os.path.exists(HIPCC):
        raise RuntimeError(f"hipcc not found ({HIPCC})")
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    srcs = SOURCES + [COPY_SOURCE]
    objs = [os.path.join(objdir, s.rsplit(".", 1)[0] + ".o") for s in srcs]
    with ThreadPoolExecutor(max_workers=min(len(srcs), os.cpu_count() or 1)) as ex:
        modules = [ex.submit(_build_table), ex.submit(_build_state_space)]
        list(ex.map(lambda so: _compile(*so), zip(srcs, objs)))
    # (the C ABI needs neither torch's headers nor Python's: it is there also where a module fails)
    _link(objs[:-1], LIB)
    _link(objs[-1:], COPY_LIB)
    for module in modules:
        module.result()
    if verbose:
        print(f"built {LIB}, {COPY_LIB}, {TABLE_LIB} and {SPACE_LIB}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
