"""Build libojx.so (the sm_100a kernels + C-ABI runtime) in-tree, and its
bounds-checking twin libojx_debug.so (-DOJX_DEBUG_BOUNDS).

    python ojasx-open-source-cuda-_b200/build.py [--verbose-ptxas]

Compiles csrc/ojx_kernels.cu (the GEMM path's kernels, one translation unit),
csrc/serving.cu (the serving operators), csrc/runtime.cpp, csrc/tmap.cpp and
csrc/graph.cpp with nvcc for `-gencode arch=compute_100a,code=sm_100a` and links
them into ojasx-open-source-cuda-_b200/torchcl/_lib/libojx.so, next to the Python
package that loads it.  The CUDA runtime is linked statically, so the library does
not depend on which libcudart another module (e.g. torch) already loaded.  Beside it
csrc/torch_binding.cpp becomes torchcl/_lib/ojx_torch.so, the serving operators' binding
for torch tensors.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import pathlib
import shutil
import subprocess
import sys

PKG = pathlib.Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
OUT_DIR = PKG / "torchcl" / "_lib"
OBJ_DIR = PKG / "_build"
LIB = OUT_DIR / "libojx.so"
BINDING = OUT_DIR / "ojx_torch.so"  # csrc/torch_binding.cpp: the serving operators on torch tensors

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3", f"-I{INCLUDE}", f"-I{CSRC}"]
SOURCES = ["ojx_kernels.cu", "serving.cu", "runtime.cpp", "tmap.cpp", "graph.cpp"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and pathlib.Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


# Two builds of the same sources: the library itself, and the bounds-checking build
# (every TMA tile origin and epilogue store checked on the device; torchcl loads it
# when OJX_DEBUG_BOUNDS=1).
VARIANTS = {"release": (LIB, OBJ_DIR, []),
            "debug": (OUT_DIR / "libojx_debug.so", OBJ_DIR / "debug", ["-DOJX_DEBUG_BOUNDS"])}


def _compile(src: str, obj_dir: pathlib.Path, defs: list[str], verbose_ptxas: bool) -> pathlib.Path:
    obj = obj_dir / (pathlib.Path(src).stem + ".o")
    cmd = [nvcc(), *ARCH, *COMMON, *defs, "-c", str(CSRC / src), "-o", str(obj)]
    if verbose_ptxas and src.endswith(".cu"):
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{res.stdout}\n{res.stderr}")
    if verbose_ptxas and res.stderr:
        (obj_dir / (pathlib.Path(src).stem + ".ptxas.txt")).write_text(res.stderr)
    return obj


def _stale(lib: pathlib.Path, deps=None) -> bool:
    if not lib.exists():
        return True
    t = lib.stat().st_mtime
    if deps is None:
        deps = [p for p in CSRC.glob("*") if p.name != "torch_binding.cpp"]
    deps = deps + list(INCLUDE.glob("*.h")) + [pathlib.Path(__file__)]
    return any(p.stat().st_mtime > t for p in deps)


def _build_binding() -> None:
    """ojx_torch.so: plain C++ against the installed torch (no CUDA code, no link to libojx)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    src = CSRC / "torch_binding.cpp"
    cuda_include = pathlib.Path(nvcc()).resolve().parents[1] / "include"
    inc = [*cpp_extension.include_paths(), str(cuda_include), sysconfig.get_paths()["include"]]
    libs = cpp_extension.library_paths()[0]
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=ojx_torch",
           "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-isystem{i}" for i in inc], str(src), "-o", str(tmp), f"-L{libs}", "-lc10", "-ltorch_cpu", "-ltorch",
           "-ltorch_python", "-lc10_cuda", f"-Wl,-rpath,{libs}"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, BINDING)


def _link(lib: pathlib.Path, objs: list[pathlib.Path]) -> None:
    tmp = lib.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-ldl"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, lib)


def build(force: bool = False, verbose_ptxas: bool = False) -> pathlib.Path:
    """Build every stale variant (both compile in parallel) and the torch binding; returns
    the release library."""
    OUT_DIR.mkdir(parents=True, exist_ok=True)
    if force or _stale(BINDING, [CSRC / "torch_binding.cpp"]):
        _build_binding()
    todo = {name: v for name, v in VARIANTS.items() if force or _stale(v[0])}
    if not todo:
        return LIB
    jobs = []
    for name, (lib, obj_dir, defs) in todo.items():
        obj_dir.mkdir(parents=True, exist_ok=True)
        jobs += [(name, src, obj_dir, defs) for src in SOURCES]
    with cf.ThreadPoolExecutor(max_workers=len(jobs)) as ex:
        objs = list(ex.map(lambda j: (j[0], _compile(j[1], j[2], j[3], verbose_ptxas)), jobs))
    for name, (lib, _, _) in todo.items():
        _link(lib, [o for n, o in objs if n == name])
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose-ptxas", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force or a.verbose_ptxas, verbose_ptxas=a.verbose_ptxas))
    sys.exit(0)
