"""Build the C-ABI shared library ``libravel_b200.so`` for sm_100a with nvcc,
and the C++ host extension ``_ravel_host`` that the Python API calls it through.

The library is plain CUDA C++ (no PyTorch headers): ``include/ravel_b200.h``
is its interface.  The host extension (``csrc/host_ext.cpp``, g++ against
PyTorch's headers) links to it.  Both are built in-tree so that they travel
with the source tree to the GPU machine.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libravel_b200.so"
OBJ = PKG / "_build"
HOST_EXT = PKG / ("_ravel_host" + sysconfig.get_config_var("EXT_SUFFIX"))

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=default",
]


def nvcc_path() -> str:
    home = os.environ.get("CUDA_HOME") or "/usr/local/cuda"
    cand = Path(home) / "bin" / "nvcc"
    if cand.exists():
        return str(cand)
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found; set CUDA_HOME")
    return found


def units() -> list[Path]:
    """The translation units of the library."""
    return sorted(CSRC.glob("*.cu"))


def includes(src: Path, seen: set[Path] | None = None) -> set[Path]:
    """``src`` and every file of this repository that it includes, directly or not."""
    seen = set() if seen is None else seen
    if src in seen:
        return seen
    seen.add(src)
    for name in re.findall(r'^\s*#include "([^"]+)"', src.read_text(), flags=re.M):
        dep = (src.parent / name).resolve()
        if dep.exists():
            includes(dep, seen)
    return seen


def host_sources() -> list[Path]:
    return [CSRC / "host_ext.cpp", ROOT / "include" / "ravel_b200.h", LIB]


def obj_path(unit: Path) -> Path:
    return OBJ / (unit.stem + ".o")


def flags_path(unit: Path) -> Path:
    return OBJ / (unit.stem + ".flags")


def compiled_with(unit: Path) -> str | None:
    """The flags of the unit's object file (None: not known)."""
    path = flags_path(unit)
    return path.read_text() if path.exists() and obj_path(unit).exists() else None


def stale(unit: Path, target: Path) -> bool:
    return not target.exists() or any(p.stat().st_mtime > target.stat().st_mtime for p in includes(unit))


def needs_build(flags: str = " ".join(NVCC_FLAGS)) -> bool:
    """Whether a source or an object is newer than the library, or an object was compiled with other flags."""
    def changed(unit: Path) -> bool:
        obj = obj_path(unit)
        unlinked = LIB.exists() and obj.exists() and obj.stat().st_mtime > LIB.stat().st_mtime
        return stale(unit, LIB) or unlinked or compiled_with(unit) not in (None, flags)
    return any(changed(u) for u in units())


def build_host(force: bool = False, verbose: bool = False) -> Path:
    """Compile ``csrc/host_ext.cpp`` into the ``_ravel_host`` extension module when it is stale."""
    if not force and HOST_EXT.exists() and all(p.stat().st_mtime <= HOST_EXT.stat().st_mtime
                                               for p in host_sources()):
        return HOST_EXT
    from torch.utils.cpp_extension import include_paths, library_paths
    cuda_inc = str(Path(os.environ.get("CUDA_HOME") or "/usr/local/cuda") / "include")
    torch_lib = library_paths()[0]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           "-DTORCH_EXTENSION_NAME=_ravel_host", "-DTORCH_API_INCLUDE_EXTENSION_H",
           *[f"-I{p}" for p in include_paths()], f"-I{cuda_inc}", f"-I{sysconfig.get_paths()['include']}",
           str(CSRC / "host_ext.cpp"), "-o", str(HOST_EXT.with_suffix(".tmp")),
           f"-L{torch_lib}", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python",
           f"-L{PKG}", "-lravel_b200", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(HOST_EXT.with_suffix(".tmp"), HOST_EXT)
    return HOST_EXT


def build(force: bool = False, verbose: bool = False, extra_flags: list[str] | None = None) -> Path:
    """Compile the stale translation units of ``csrc`` (in parallel) and link ``libravel_b200.so``, then build
    the host extension."""
    flags = " ".join([*NVCC_FLAGS, *(extra_flags or [])])
    if not force and not needs_build(flags):
        build_host(force=force, verbose=verbose)
        return LIB
    OBJ.mkdir(exist_ok=True)

    def compile_unit(unit: Path) -> None:
        obj = obj_path(unit)
        tmp = obj.with_suffix(".o.tmp")
        cmd = [nvcc_path(), *NVCC_FLAGS, *(extra_flags or []), "-c", "-o", str(tmp), str(unit)]
        if verbose:
            print(" ".join(cmd), flush=True)
        flags_path(unit).unlink(missing_ok=True)
        subprocess.run(cmd, check=True)
        os.replace(tmp, obj)
        flags_path(unit).write_text(flags)

    todo = [u for u in units() if force or stale(u, obj_path(u)) or compiled_with(u) != flags]
    with ThreadPoolExecutor(max_workers=max(1, len(todo))) as pool:
        list(pool.map(compile_unit, todo))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc_path(), *NVCC_FLAGS, "-shared", "-o", str(tmp), *(str(obj_path(u)) for u in units())]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    build_host(force=True, verbose=verbose)
    return LIB


if __name__ == "__main__":
    build(force=True, verbose=True)
    print(LIB)
