"""In-tree build of libspecb200.so (the CUDA kernels + C ABI) for sm_100a, and of _torch_ops.so, the
extension module through which specb200.ops calls the 8-bit operators with torch tensors.

    python -m specb200.build        (with speculative-decoder_b200/ on sys.path)

Each .cu file under csrc/ is compiled to an object in parallel, then linked into
specb200/libspecb200.so next to this file, so the library travels with the source tree.
Rebuilds only when a source or header is newer than the library.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = ROOT / "csrc"
INCLUDE = ROOT.parent / "include"
LIB = PKG / "libspecb200.so"
TORCH_OPS_SRC = CSRC / "torch_ops.cpp"
TORCH_OPS = PKG / "_torch_ops.so"
OBJ_DIR = PKG / "_obj"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wno-unused-function",
         "-diag-suppress", "550,177"]


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found: the CUDA 12.9 toolkit is required to build libspecb200.so")
    return found


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _inputs() -> list[Path]:
    return _sources() + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def up_to_date() -> bool:
    if not LIB.exists():
        return False
    built = LIB.stat().st_mtime
    return all(p.stat().st_mtime <= built for p in _inputs())


def _run(cmd: list[str], what: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{res.stdout}\n{res.stderr}")


def torch_ops_target() -> str:
    """What the extension module is compiled for: it uses torch's C++ classes and Python's C API."""
    import torch

    return (f"torch {torch.__version__}, C++11 ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, "
            f"Python {sys.version_info.major}.{sys.version_info.minor}")


def _torch_ops_up_to_date() -> bool:
    stamp = TORCH_OPS.with_suffix(".stamp")
    if not TORCH_OPS.exists() or not stamp.exists() or stamp.read_text() != torch_ops_target():
        return False
    built = TORCH_OPS.stat().st_mtime
    return all(p.stat().st_mtime <= built for p in (TORCH_OPS_SRC, INCLUDE / "specb200.h"))


def build_torch_ops(verbose: bool = False, force: bool = False) -> Path:
    """The extension module, linked to libspecb200.so beside it and to the installed torch. A stamp beside it
    says what it was built for, so that another torch or Python builds it again."""
    if not force and _torch_ops_up_to_date():
        return TORCH_OPS
    import sysconfig

    import torch

    gxx = shutil.which("g++")
    if gxx is None:
        raise RuntimeError("g++ not found: the 8-bit operators of specb200.ops need _torch_ops.so (libspecb200.so is built)")
    base = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = TORCH_OPS.with_suffix(".so.tmp")
    _run([gxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DSPECB200_TARGET="{torch_ops_target()}"',
          *(f"-I{p}" for p in (INCLUDE, sysconfig.get_paths()["include"], cuda / "include")),
          *(f"-isystem{p}" for p in (base / "include", base / "include" / "torch" / "csrc" / "api" / "include")),
          str(TORCH_OPS_SRC), "-o", str(tmp), f"-L{PKG}", "-l:libspecb200.so", f"-L{base / 'lib'}", "-lc10", "-lc10_cuda",
          "-ltorch_cpu", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN"], "_torch_ops (the 8-bit operators of specb200.ops; libspecb200.so is built)",
         verbose)
    os.replace(tmp, TORCH_OPS)
    TORCH_OPS.with_suffix(".stamp").write_text(torch_ops_target())
    return TORCH_OPS


def build(verbose: bool = False, force: bool = False) -> Path:
    build_lib(verbose, force)
    build_torch_ops(verbose, force)
    return LIB


def build_lib(verbose: bool = False, force: bool = False) -> Path:
    if not force and up_to_date():
        return LIB
    OBJ_DIR.mkdir(exist_ok=True)
    cc = nvcc()

    def compile_one(src: Path) -> Path:
        obj = OBJ_DIR / (src.stem + ".o")
        cmd = [cc, *ARCH, *FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
        return obj

    with ThreadPoolExecutor(max_workers=max(1, min(8, os.cpu_count() or 1))) as pool:
        objs = list(pool.map(compile_one, _sources()))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [cc, *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-lcudart_static", "-ldl", "-lrt", "-lpthread"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
