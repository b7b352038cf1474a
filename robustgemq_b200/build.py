"""Build ``libgemq_b200.so`` in-tree for sm_100a with nvcc.

The library has no libcuda link dependency (the TMA descriptor encoder is fetched
through ``cudaGetDriverEntryPoint``) and links the CUDA runtime statically, so it
loads on machines without a GPU driver (the CPU tests check its exported symbols).

    python -m robustgemq_b200.build [--force] [--verbose]
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libgemq_b200.so"
SOURCES = ["gemq_api.cu", "kernels_misc.cu", "kernels_route.cu", "kernels_decode.cu", "kernels_tc.cu",
           "kernels_tcd.cu", "kernels_simt.cu", "kernels_cache.cu", "kernels_attn.cu", "kernels_attn_tc.cu", "kernels_verify.cu",
           "serving_api.cu"]
# the torch binding of the serving operators
EXT = PKG / "_serving_ext.so"
EXT_SOURCE = "serving_ext.cpp"
EXT_STAMP = ROOT / "_build" / "serving_ext.torch"  # the torch version it was compiled with
HEADERS = ["gemq_common.cuh", "gemq_internal.h", "tc_work.cuh", "kperm.cuh", "paged.cuh", "attn_rows.cuh"]
# compiled without relocatable device code: ptxas ignores setmaxnreg with it
WHOLE = {"kernels_attn_tc.cu"}
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _stale() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = [CSRC / s for s in SOURCES + HEADERS] + [ROOT / "include" / "gemq_b200.h"]
    return any(p.stat().st_mtime > t for p in deps)


def _ext_stale() -> bool:
    if not EXT.exists():
        return True
    if EXT_STAMP.exists() and EXT_STAMP.read_text() != _torch_version():
        return True  # another torch's headers
    t = EXT.stat().st_mtime
    return any(p.stat().st_mtime > t for p in (CSRC / EXT_SOURCE, ROOT / "include" / "gemq_b200.h"))


def _torch_version() -> str:
    import torch

    return torch.__version__


def _ext_commands(obj: Path):
    """Compile and link commands of the torch binding (host code only)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    includes = [*cpp_extension.include_paths(device_type="cuda"), sysconfig.get_paths()["include"]]
    compile_cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                   "-DTORCH_EXTENSION_NAME=_serving_ext", *[f"-I{p}" for p in includes], "-c", str(CSRC / EXT_SOURCE),
                   "-o", str(obj)]
    libs = [f"-L{p}" for p in cpp_extension.library_paths()]
    link_cmd = ["g++", "-shared", "-o", str(EXT.with_suffix(".so.tmp")), str(obj), f"-L{PKG}", "-l:libgemq_b200.so",
                "-Wl,-rpath,$ORIGIN", *libs, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    return compile_cmd, link_cmd


def build(force: bool = False, verbose: bool = False, jobs: int = 4) -> Path:
    """Builds the library and, beside it, the torch binding of the serving operators. The
    library does not need the binding: it is built before what stops that is raised."""
    ext, failed = None, None
    if force or _ext_stale():
        try:
            ext = _start_ext()
        except Exception as exc:  # no g++, no Python headers
            failed = exc
    build_library(force, verbose, jobs)
    if failed is not None:
        raise RuntimeError(f"the torch binding could not be built: {failed}") from failed
    if ext is not None:
        _finish_ext(ext, verbose)
    return LIB


def build_library(force: bool = False, verbose: bool = False, jobs: int = 4) -> Path:
    """Builds the library where its sources are newer."""
    if force or _stale():
        _build_lib(verbose, jobs)
    return LIB


def build_binding(verbose: bool = False) -> Path:
    """Builds the torch binding (beside a library that is there) where its sources are
    newer or torch is another."""
    if _ext_stale():
        _finish_ext(_start_ext(), verbose)
    return EXT


def _start_ext():
    objdir = ROOT / "_build"
    objdir.mkdir(exist_ok=True)
    compile_cmd, link_cmd = _ext_commands(objdir / "serving_ext.o")
    return subprocess.Popen(compile_cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True), link_cmd


def _finish_ext(ext, verbose: bool) -> None:
    proc, link_cmd = ext
    _wait((EXT_SOURCE, proc), verbose)
    out = subprocess.run(link_cmd, capture_output=True, text=True)
    if out.returncode != 0:
        raise RuntimeError(f"link failed:\n{out.stdout}\n{out.stderr}")
    os.replace(EXT.with_suffix(".so.tmp"), EXT)
    EXT_STAMP.write_text(_torch_version())


def _build_lib(verbose: bool, jobs: int) -> Path:
    nvcc = nvcc_path()
    objdir = ROOT / "_build"
    objdir.mkdir(exist_ok=True)
    common = [nvcc, *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I", str(ROOT / "include"),
              "--expt-relaxed-constexpr"]
    if verbose:
        common += ["-Xptxas", "-v"]
    procs = []
    objs = []
    for src in SOURCES:
        obj = objdir / (Path(src).stem + ".o")
        objs.append(obj)
        cmd = common + ([] if src in WHOLE else ["-rdc=true"]) + ["-c", str(CSRC / src), "-o", str(obj)]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        if len(procs) >= jobs:
            _wait(procs.pop(0), verbose)
    for p in procs:
        _wait(p, verbose)
    tmp = LIB.with_suffix(".so.tmp")
    link = [nvcc, *ARCH, "-shared", "-rdc=true", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
    out = subprocess.run(link, capture_output=True, text=True)
    if out.returncode != 0:
        raise RuntimeError(f"link failed:\n{out.stdout}\n{out.stderr}")
    os.replace(tmp, LIB)
    return LIB


def _wait(item, verbose):
    src, proc = item
    out, _ = proc.communicate()
    if proc.returncode != 0:
        raise RuntimeError(f"compiler failed on {src}:\n{out}")
    if verbose and out:
        sys.stdout.write(f"--- {src}\n{out}")


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
