"""Builds libsvl_b200.so (the sm_100a kernels and the C ABI) in-tree with nvcc, and the operators'
binding to torch tensors (svl/_torch_ops.so) with the host compiler.

Run `python semantic-ai_b200/build.py` or call build(). Objects go to semantic-ai_b200/_build/,
the library to semantic-ai_b200/libsvl_b200.so. Only sources newer than their object are
recompiled.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OUT = PKG / "_build"
LIB = PKG / "libsvl_b200.so"
TORCH_SRC = CSRC / "torch_ops.cpp"
TORCH_OPS = PKG / "svl" / "_torch_ops.so"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

# -fmad=false: no implicit a*b+c contraction, so element-wise arithmetic rounds like the
# reference CPU path; kernels request FMAs with fmaf() where they want them.
NVCC_FLAGS = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-fmad=false", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-fvisibility=hidden,-O3",
    "-I", str(PKG.parent / "include"),
]


def _sources():
    return sorted(CSRC.glob("*.cu"))


def _deps():
    return list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + [PKG.parent / "include" / "svl_cuda.h"]


def _compile(src: Path, extra: list[str]) -> Path:
    obj = OUT / (src.stem + ".o")
    newest_dep = max([src.stat().st_mtime] + [d.stat().st_mtime for d in _deps()])
    if obj.exists() and obj.stat().st_mtime >= newest_dep:
        return obj
    cmd = [NVCC, *NVCC_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    if r.stderr.strip():
        sys.stderr.write(r.stderr)
    return obj


def _built_for() -> str | None:
    """What the binding has to match besides its sources: torch, its C++ ABI and Python's. None without torch."""
    import sysconfig

    try:
        import torch
    except ImportError:
        return None
    return f"torch {torch.__version__} cxx11 {int(torch._C._GLIBCXX_USE_CXX11_ABI)} {sysconfig.get_config_var('EXT_SUFFIX')}"


def _build_torch_ops() -> None:
    key, stamp = _built_for(), OUT / "torch_ops.stamp"
    if key is None:
        sys.stderr.write(f"{TORCH_OPS.name} is not built: torch cannot be imported\n")
        return
    newest = max(TORCH_SRC.stat().st_mtime, (PKG.parent / "include" / "svl_cuda.h").stat().st_mtime)
    if TORCH_OPS.exists() and TORCH_OPS.stat().st_mtime >= newest and stamp.exists() and stamp.read_text() == key:
        return
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    # nvcc's own host compiler, as for the library: another one's C++ library may not be torch's.
    cmd = [NVCC, "-std=c++17", "-O2", "-shared", "-cudart", "none", "-Xcompiler", "-fPIC,-fvisibility=hidden,-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", str(root / "include"), "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", sysconfig.get_paths()["include"], str(TORCH_SRC), "-o", str(TORCH_OPS),
           "-L", str(root / "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"building {TORCH_OPS.name} failed:\n{r.stdout}\n{r.stderr}")
    stamp.write_text(key)


def build(verbose: bool = False, extra: list[str] | None = None) -> Path:
    """The library and, where torch can be imported, the binding, whose failure leaves the library built."""
    OUT.mkdir(exist_ok=True)
    extra = extra or []
    with cf.ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as ex:
        ops = ex.submit(_build_torch_ops)
        objs = list(ex.map(lambda s: _compile(s, extra), _sources()))
    _link(objs, verbose)
    ops.result()
    return LIB


def _link(objs: list[Path], verbose: bool) -> None:
    if LIB.exists() and LIB.stat().st_mtime >= max(o.stat().st_mtime for o in objs):
        return
    cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a",
           "-Xcompiler", "-fPIC", "-o", str(LIB), *map(str, objs), "-cudart", "static"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(f"built {LIB}")


if __name__ == "__main__":
    extra = sys.argv[1:]
    build(verbose=True, extra=extra)
