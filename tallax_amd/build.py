"""Build the gfx950 HIP library `tallax_amd/_build/libtallax_hip.so` and the
Python module `tallax_amd/_build/serving_ext.so` that calls it.

One hipcc invocation per source (parallel), then one link.  Every HIP source is
compiled with:
  * --offload-arch=gfx950 (MI355X only);
  * -ffp-contract=off, so every float operation on the sampler path is a single
    IEEE binary32 operation that the numpy oracle reproduces bit for bit;
  * -Xclang -target-feature -Xclang -packed-fp32-ops, which keeps the compiler
    from emitting packed-FP32 VALU instructions.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import pathlib
import shutil
import subprocess
import sys
import sysconfig

PKG = pathlib.Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OUT_DIR = PKG / "_build"
LIB_NAME = "libtallax_hip.so"
LIB_PATH = OUT_DIR / LIB_NAME
EXT_SOURCE = "serving_ext.cpp"  # host code: between torch tensors and the library's C ABI
EXT_PATH = OUT_DIR / "serving_ext.so"

SOURCES = [
    "capi.hip",
    "row_select.hip",
    "topk_short.hip",
    "scan_gather.hip",
    "sort_rows.hip",
    "sort_wide.hip",
    "binned.hip",
    "softmax_topk.hip",
    "sample_wide.hip",
    "kv_cache.hip",
    "kv_attention.hip",
    "kv_rotate.hip",
    "kv_shared.hip",
    "route.hip",
    "verify.hip",
    "testing.hip",
]

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

COMMON_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-function",
    "-Wno-unused-variable",
    f"-I{CSRC}",
    f"-I{PKG.parent / 'include'}",
]


def _compile(src: str, obj_dir: pathlib.Path) -> pathlib.Path:
    obj = obj_dir / (pathlib.Path(src).stem + ".o")
    cmd = [HIPCC, *COMMON_FLAGS, "-c", str(CSRC / src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")
    return obj


def _compile_ext(obj_dir: pathlib.Path) -> pathlib.Path:
    import torch

    obj = obj_dir / "serving_ext.o"
    root = pathlib.Path(torch.__file__).parent
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-I{root / 'include'}",
           f"-I{pathlib.Path(HIPCC).resolve().parent.parent / 'include'}", f"-I{sysconfig.get_paths()['include']}",
           f"-I{PKG.parent / 'include'}", "-c", str(CSRC / EXT_SOURCE), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed for {EXT_SOURCE}:\n{' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")
    return obj


def _link_ext(obj: pathlib.Path) -> None:
    import torch

    tmp = OUT_DIR / (EXT_PATH.name + ".tmp")
    cmd = ["g++", "-shared", "-fPIC", str(obj), f"-L{OUT_DIR}", f"-l:{LIB_NAME}", "-Wl,-rpath,$ORIGIN",
           f"-L{pathlib.Path(torch.__file__).parent / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_hip",
           "-Wl,--allow-shlib-undefined", "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, EXT_PATH)


def build(verbose: bool = True) -> pathlib.Path:
    """Compile every HIP source for gfx950, link the shared library and the Python module over it."""
    if shutil.which(HIPCC) is None and not os.path.exists(HIPCC):
        raise RuntimeError(f"hipcc not found at {HIPCC}")
    OUT_DIR.mkdir(exist_ok=True)
    obj_dir = OUT_DIR / "obj"
    obj_dir.mkdir(exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(8, len(SOURCES))) as ex:
        ext = ex.submit(_compile_ext, obj_dir)
        objs = list(ex.map(lambda s: _compile(s, obj_dir), SOURCES))
        ext = ext.result()
    tmp = OUT_DIR / (LIB_NAME + ".tmp")
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, LIB_PATH)
    _link_ext(ext)
    if verbose:
        print(f"built {LIB_PATH} and {EXT_PATH.name}", file=sys.stderr)
    return LIB_PATH


if __name__ == "__main__":
    build()
