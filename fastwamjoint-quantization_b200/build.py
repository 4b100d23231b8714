"""Build ``libsq_b200.so`` in-tree with nvcc for sm_100a.

    python fastwamjoint-quantization_b200/build.py [--force] [--verbose]

The library has a C ABI only (``include/sq_b200.h``); it links the CUDA runtime
statically and needs neither PyTorch nor libcuda at link time (the one driver
call it makes, ``cuTensorMapEncodeTiled``, is looked up at run time).

Beside it goes ``sq_binding``, a small CPython module over that C ABI which takes the
block operators' ordinary calls (``csrc/sq_binding.cpp``); it is compiled by the host
compiler against PyTorch's headers.  It is optional: where it cannot be built there is a
warning, and the calls go through ctypes.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
LIB = HERE / "lib" / "libsq_b200.so"
BINDING_SOURCE = CSRC / "sq_binding.cpp"
SOURCES = ("sq_prepass.cu", "sq_gemm_tc.cu", "sq_gemm_ts.cu", "sq_fp8_gemm.cu", "sq_block_norm.cu", "sq_rotary.cu",
           "sq_api.cu")
HEADERS = ("sq_internal.h", "sq_overlap.h", "sq_ptx.cuh", "sq_rows.cuh", "../../include/sq_b200.h")
NVCC_FLAGS = ("-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden")


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found; libsq_b200.so cannot be built.")
    return found


def stale() -> bool:
    if not LIB.exists():
        return True
    built = LIB.stat().st_mtime
    deps = [CSRC / s for s in SOURCES] + [(CSRC / h).resolve() for h in HEADERS] + [Path(__file__)]
    return any(d.stat().st_mtime > built for d in deps)


def binding_path() -> Path | None:
    """Where the binding for this interpreter and this PyTorch lies, or None without a PyTorch.  The module reads C++ objects
    of both, so its name says which it was compiled against: another release finds no module, not a wrong one."""
    spec = importlib.util.find_spec("torch")
    version = Path(spec.origin).with_name("version.py") if spec is not None and spec.origin else None
    found = re.search(r"^__version__ = '([^']+)'", version.read_text(), re.M) if version is not None and version.exists() else None
    if found is None:
        return None
    return LIB.with_name(f"sq_binding.{sysconfig.get_config_var('SOABI')}.torch-{found[1]}.so")


def build_binding(force: bool = False, verbose: bool = False) -> Path | None:
    """The binding, linked against the built library (found beside it at run time) and PyTorch's own; None, with a warning,
    where it cannot be built."""
    binding, compiler = binding_path(), shutil.which("g++")
    if binding is None or compiler is None:
        warnings.warn("sq_binding needs PyTorch and g++ to be built; the block operators' calls go through ctypes.")
        return None
    deps = [BINDING_SOURCE, (CSRC / "../../include/sq_b200.h").resolve(), Path(__file__)]
    if not force and binding.exists() and all(d.stat().st_mtime <= binding.stat().st_mtime for d in deps):
        return binding
    torch_dir = Path(importlib.util.find_spec("torch").origin).parent
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = binding.with_suffix(".so.tmp")
    cmd = [compiler, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-isystem", str(torch_dir / "include"),
           "-isystem", str(torch_dir / "include/torch/csrc/api/include"), "-isystem", str(cuda / "include"),
           "-I", sysconfig.get_paths()["include"], str(BINDING_SOURCE), "-o", str(tmp), f"-L{LIB.parent}", f"-l:{LIB.name}",
           f"-L{torch_dir / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10", "-Wl,-rpath,$ORIGIN"]
    done = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or done.returncode:
        sys.stderr.write(done.stdout + done.stderr)
    if done.returncode:
        binding.unlink(missing_ok=True)  # of older sources
        warnings.warn("building sq_binding failed; the block operators' calls go through ctypes.")
        return None
    os.replace(tmp, binding)
    return binding


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not stale():
        build_binding(verbose=verbose)
        return LIB
    obj_dir = HERE / "build"
    obj_dir.mkdir(exist_ok=True)
    LIB.parent.mkdir(exist_ok=True)
    compiler = nvcc()

    def compile_one(source: str) -> Path:
        obj = obj_dir / (source + ".o")
        cmd = [compiler, *NVCC_FLAGS, "-c", str(CSRC / source), "-o", str(obj)]
        if verbose:
            cmd += ["-Xptxas", "-v"]
            print(" ".join(cmd), flush=True)
        done = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or done.returncode:
            sys.stderr.write(done.stdout + done.stderr)
        if done.returncode:
            raise RuntimeError(f"nvcc failed on {source}")
        return obj

    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 1)) as pool:
        objects = list(pool.map(compile_one, SOURCES))
    tmp = LIB.with_suffix(".so.tmp")
    link = [compiler, "-shared", "-o", str(tmp), *map(str, objects), "-cudart", "static",
            "-gencode", "arch=compute_100a,code=sm_100a"]
    done = subprocess.run(link, capture_output=True, text=True)
    if done.returncode:
        sys.stderr.write(done.stdout + done.stderr)
        raise RuntimeError("linking libsq_b200.so failed")
    os.replace(tmp, LIB)
    build_binding(force=force, verbose=verbose)
    return LIB


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--verbose", action="store_true")
    args = parser.parse_args()
    print(build(force=args.force, verbose=args.verbose))
