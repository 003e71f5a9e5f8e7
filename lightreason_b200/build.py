"""Build libmoe_b200.so in-tree with nvcc for sm_100a.

The shared library is the product's native half: every CUDA kernel and the C
ABI declared in include/moe_b200.h.  It is built next to this file
(lightreason_b200/_native/) so that it travels with the source tree, and with
it _fp8_bind, the Python module through which the FP8 entry points call it.
The module needs a host C++ compiler, Python's headers and torch's, and is bound
to one torch (its version is in the file's name); where it cannot be built, the
library still is, and the FP8 entry points of Python say what is missing.
"""

from __future__ import annotations

import importlib.metadata
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OUT_DIR = PKG / "_native"
LIB = OUT_DIR / "libmoe_b200.so"
SOURCES = ["host.cu", "router.cu", "permute.cu", "experts.cu", "layer.cu", "gather.cu", "grouped.cu",
           "expert_rows_noalloc.cu", "expert_parallel.cu", "router_tc.cu", "primary.cu", "ep_p2p.cu",
           "codec.cu", "decode.cu", "fp8_quant.cu", "fp8_gemv.cu", "fp8_tc.cu", "fp8_api.cu"]


def _torch_version() -> str:
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return "none"


BIND = OUT_DIR / f"_fp8_bind.torch-{_torch_version()}{sysconfig.get_config_var('EXT_SUFFIX') or '.so'}"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libmoe_b200.so")
    return cand


def _older(built: Path, deps) -> bool:
    return not built.exists() or any(p.stat().st_mtime > built.stat().st_mtime for p in deps if p.exists())


def _lib_stale() -> bool:
    return _older(LIB, [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + [ROOT / "include" / "moe_b200.h"])


def _bind_stale() -> bool:
    return _older(BIND, [CSRC / "fp8_bind.cpp", ROOT / "include" / "moe_b200.h"])


def _bind_command(out: Path) -> list[str]:
    """The host compiler's line for the Python module: torch's headers and
    libraries (which are loaded wherever the module is)."""
    import torch

    home = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1]
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    return [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
            "-I", str(ROOT / "include"), "-isystem", str(home / "include"),
            "-isystem", str(home / "include" / "torch" / "csrc" / "api" / "include"),
            "-isystem", sysconfig.get_paths()["include"], "-isystem", str(cuda / "include"),
            str(CSRC / "fp8_bind.cpp"), "-o", str(out), "-L", str(home / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
            "-ltorch_python"]


def _build_lib(verbose: bool) -> None:
    """Compile every .cu in csrc/ for sm_100a and link libmoe_b200.so."""
    obj_dir = OUT_DIR / "obj"
    obj_dir.mkdir(exist_ok=True)
    flags = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I", str(ROOT / "include"),
                    "-I", str(CSRC), "--expt-relaxed-constexpr"]
    if verbose:
        flags += ["-Xptxas", "-v"]
    objs, procs = [], []
    for src in SOURCES:
        obj = obj_dir / (Path(src).stem + ".o")
        objs.append(obj)
        cmd = [nvcc(), *flags, "-c", str(CSRC / src), "-o", str(obj)]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = []
    for src, proc in procs:
        out, _ = proc.communicate()
        if verbose or proc.returncode:
            sys.stderr.write(out)
        if proc.returncode:
            failed.append(src)
    if failed:
        raise RuntimeError(f"nvcc failed for {failed}")
    tmp = LIB.with_suffix(".so.tmp")
    subprocess.run([nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs),], check=True)
    os.replace(tmp, LIB)


def _build_bind(verbose: bool) -> None:
    """Compile _fp8_bind.  Callers of the C ABI and of the BF16 layer do without
    it, so a machine that cannot (no host compiler, headers or torch) is told."""
    tmp = BIND.with_name(BIND.name + ".tmp")
    try:
        done = subprocess.run(_bind_command(tmp), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        out, failed = done.stdout, done.returncode != 0
    except (OSError, ImportError) as error:
        out, failed = f"{error}\n", True
    if verbose or failed:
        sys.stderr.write(out)
    if failed:
        sys.stderr.write(f"{BIND.name} was not built: the FP8 entry points of Python are not available\n")
    else:
        os.replace(tmp, BIND)


def build(force: bool = False, verbose: bool = False, jobs: int = 0) -> Path:
    """libmoe_b200.so and _fp8_bind, those of them that are not up to date."""
    lib, bind = force or _lib_stale(), force or _bind_stale()
    if lib or bind:
        OUT_DIR.mkdir(exist_ok=True)
    with ThreadPoolExecutor(1) as side:
        module = side.submit(_build_bind, verbose) if bind else None
        if lib:
            _build_lib(verbose)
        if module:
            module.result()
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
