"""Builds libd3moe.so (every CUDA source under csrc/) for sm_100a with nvcc, and the
CPython binding _d3native.so (csrc/binding/) with g++.

The libraries are written in-tree next to the Python package (d3moe/_lib/) so
that they travel with the source tree; they are rebuilt only when a source or
header is newer than they are, the binding also when the installed torch is not
the one it was built for. Without torch libd3moe.so is built alone: it needs
nvcc only, the binding g++ and torch as well.

Usage: python build.py [--force] [--verbose]
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OUT_DIR = HERE / "d3moe" / "_lib"
LIB = OUT_DIR / "libd3moe.so"
# test-only library (csrc/selftest/): failure-path probes kept out of the product
SELFTEST_LIB = OUT_DIR / "libd3moe_selftest.so"
# CPython binding of the operators whose host time counts (csrc/binding/)
NATIVE_LIB = OUT_DIR / "_d3native.so"
INCLUDE = HERE.parent / "include"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler",
    "-fPIC,-fvisibility=hidden",
    "-Xptxas",
    "-warn-spills",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; the CUDA 12.9 toolkit is required to build libd3moe.so")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def torch_version() -> str | None:
    """Version of the installed torch (without importing it), None when there is none."""
    import importlib.metadata

    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return None


def binding_mark(version: str | None) -> str:
    """The text by which the binding says which torch it was built for."""
    return f"d3moe binding for torch {version};"


def _older(built: tuple[Path, ...], sources: list[Path]) -> bool:
    if not all(p.exists() for p in built):
        return True
    lib_time = min(p.stat().st_mtime for p in built)
    deps = sources + list(INCLUDE.glob("*.h")) + [Path(__file__)]
    return any(p.stat().st_mtime > lib_time for p in deps if p.is_file())


def library_needs_build() -> bool:
    return _older((LIB, SELFTEST_LIB), [p for p in CSRC.rglob("*") if p.parent.name != "binding"])


def binding_needs_build() -> bool:
    version = torch_version()
    if version is None:
        return False
    return _older((NATIVE_LIB,), list((CSRC / "binding").glob("*"))) or binding_mark(version).encode() not in NATIVE_LIB.read_bytes()


def needs_build() -> bool:
    return library_needs_build() or binding_needs_build()


def _link(cc: str, srcs: list[Path], out: Path, objdir: Path, verbose: bool) -> None:
    objs = []
    for src in srcs:
        obj = objdir / (src.stem + ".o")
        cmd = [cc, *ARCH_FLAGS, *NVCC_FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
        if verbose:
            cmd += ["-Xptxas", "-v"]
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        objs.append(str(obj))
    tmp = out.with_suffix(".so.tmp")
    cmd = [cc, *ARCH_FLAGS, "-shared", "-Xlinker", "--no-undefined", "-o", str(tmp), *objs, "-lcudart"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, out)


def _link_binding(out: Path, verbose: bool) -> None:
    """The CPython binding, against torch's headers and libraries."""
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    cxx = os.environ.get("CXX") or shutil.which("g++")
    if not cxx:
        raise RuntimeError("g++ not found; it compiles the CPython binding")
    cuda = Path(nvcc()).resolve().parents[1]
    include = [INCLUDE, root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
               cuda / "include", Path(sysconfig.get_paths()["include"])]
    tmp = out.with_suffix(".so.tmp")
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f'-DD3_BUILT_FOR="{binding_mark(torch_version())}"',
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *[f"-I{p}" for p in include], *map(str, sorted((CSRC / "binding").glob("*.cpp"))), "-o", str(tmp),
           f"-L{root / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, out)


def build(force: bool = False, verbose: bool = False) -> Path:
    library = force or library_needs_build()
    OUT_DIR.mkdir(parents=True, exist_ok=True)
    objdir = HERE / "_build"
    objdir.mkdir(exist_ok=True)
    if library:
        cc = nvcc()
        _link(cc, sources(), LIB, objdir, verbose)
        _link(cc, sorted((CSRC / "selftest").glob("*.cu")), SELFTEST_LIB, objdir, verbose)
    if torch_version() is None:
        print("torch is not installed: the CPython binding of the sequence-memory operators is left out", file=sys.stderr)
    elif force or binding_needs_build():
        _link_binding(NATIVE_LIB, verbose)
    return LIB


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
    return 0


if __name__ == "__main__":
    sys.exit(main())
