"""Build the sm_100a shared library in-tree with nvcc.

The library is self-contained (static CUDA runtime) and is written next to this
file as ``libkernix_b200.so`` so that it travels with the source tree.  The
binding of the Python mirror's calls on torch tensors, which knows torch and
nothing of CUDA, is written beside it as ``_kx_torch`` with the interpreter's
suffix; without torch it is left out, and the C ABI is all there is.
"""
from __future__ import annotations

import importlib.util
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OBJ = ROOT / "_build" / "kernix_b200"
LIB = PKG / "libkernix_b200.so"
BINDING = PKG / ("_kx_torch" + sysconfig.get_config_var("EXT_SUFFIX"))

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
         "-I", str(ROOT / "include")]


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.hpp")) + sorted((ROOT / "include").glob("*.h"))


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _compile(src: Path, verbose: bool) -> Path:
    obj = OBJ / (src.stem + ".o")
    if _stale(obj, [src] + _headers()):
        cmd = [NVCC, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
    return obj


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every CUDA source for sm_100a and link libkernix_b200.so."""
    OBJ.mkdir(parents=True, exist_ok=True)
    srcs = _sources()
    if force:
        for o in OBJ.glob("*.o"):
            o.unlink()
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    if force or _stale(LIB, objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [NVCC, *ARCH, "-shared", "-o", str(tmp), *map(str, objs)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIB)
    _binding(force, verbose)
    return LIB


def _binding(force: bool, verbose: bool) -> None:
    """Compile csrc/kx_torch.cpp against the installed torch; again where that
    is another one than the last time, whatever its files' times."""
    src = CSRC / "kx_torch.cpp"
    spec = importlib.util.find_spec("torch")
    torch = Path(spec.submodule_search_locations[0]) if spec else None
    if torch is None or not (torch / "include" / "ATen" / "ATen.h").exists():
        print("kernix_b200: no torch with its headers: the Python binding is left out", file=sys.stderr)
        return
    built_for, this = OBJ / "binding.txt", f"{torch}\n{(torch / 'version.py').read_text()}"
    same = built_for.exists() and built_for.read_text() == this
    if not force and same and not _stale(BINDING, [src] + _headers()):
        return
    (PKG / "_kx_torch.so").unlink(missing_ok=True)      # of any interpreter, as it was named once
    built_for.unlink(missing_ok=True)
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-Wall", "-shared", "-fPIC", "-fvisibility=hidden",
           "-I", sysconfig.get_paths()["include"], "-isystem", str(torch / "include"), "-isystem",
           str(torch / "include" / "torch" / "csrc" / "api" / "include"), str(src), "-o", str(tmp),
           "-L", str(torch / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING)
    built_for.write_text(this)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
