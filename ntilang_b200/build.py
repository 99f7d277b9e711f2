"""Build libntl_kernels.so in-tree with nvcc for sm_100a.

``python -m ntilang_b200.build`` (or ``__graft_entry__.build()``) compiles every
``csrc/*.cu`` to an object under ``ntilang_b200/_build/`` and links
``ntilang_b200/libntl_kernels.so``.  The library is plain C ABI (``include/ntl_kernels.h``);
Python reaches it through ctypes (``ntilang_b200._lib``).  Where a torch built for CUDA is installed it also builds
``csrc/paged_binding.cpp`` into ``ntilang_b200/_paged.so``, the module behind ``ntilang_b200.paged``.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libntl_kernels.so"
BINDING = PKG / "_paged.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
              "--expt-relaxed-constexpr", f"-I{ROOT / 'include'}"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; install the CUDA toolkit or set NVCC")


def sources():
    return sorted(CSRC.glob("*.cu"))


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _torch_build() -> tuple[str, str | None] | None:
    """Version of the torch that would be imported, and of its CUDA (None: built without); None where there is no
    torch.  Read from ``torch/version.py``: importing torch takes seconds."""
    import importlib.util
    import runpy

    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        return None
    version = runpy.run_path(str(Path(spec.origin).parent / "version.py"))
    return version["__version__"], version.get("cuda")


def build_binding(force: bool = False, verbose: bool = False) -> Path | None:
    """``_paged.so``, linked to the library and to torch's; None where there is no torch built for CUDA."""
    import sysconfig

    torch_build = _torch_build()
    if torch_build is None or torch_build[1] is None:
        return None
    src = CSRC / "paged_binding.cpp"
    # What it was built for; another torch or interpreter needs its own.
    note, built_for = BUILD / "_paged.torch", f"{torch_build[0]} {sysconfig.get_config_var('SOABI')}"
    if (not force and not _stale(BINDING, [src, ROOT / "include" / "ntl_kernels.h", Path(__file__)])
            and note.exists() and note.read_text() == built_for):
        return BINDING
    import torch
    from torch.utils.cpp_extension import include_paths

    cuda = Path(nvcc_path()).resolve().parents[1]
    lib = Path(torch.__file__).parent / "lib"
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-I{sysconfig.get_paths()['include']}",
           *(f"-isystem{p}" for p in include_paths()), f"-isystem{cuda / 'include'}", str(src), "-o", str(tmp),
           f"-L{PKG}", "-l:libntl_kernels.so", f"-L{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("building _paged.so failed:\n" + res.stdout + res.stderr)
    os.replace(tmp, BINDING)
    BUILD.mkdir(exist_ok=True)
    note.write_text(built_for)
    return BINDING


def build_library(force: bool = False, verbose: bool = False) -> Path:
    headers = list(CSRC.glob("*.cuh")) + [ROOT / "include" / "ntl_kernels.h"]
    srcs = sources()
    if not force and not _stale(LIB, srcs + headers + [Path(__file__)]):
        build_binding(verbose=verbose)
        return LIB
    nvcc = nvcc_path()
    BUILD.mkdir(exist_ok=True)
    procs = []
    objects = []
    for src in srcs:
        obj = BUILD / (src.stem + ".o")
        objects.append(obj)
        if not force and not _stale(obj, [src] + headers):
            continue
        cmd = [nvcc, *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failures = []
    for src, proc in procs:
        out, _ = proc.communicate()
        if proc.returncode != 0:
            failures.append(f"{src.name}:\n{out}")
        elif verbose and out.strip():
            print(out, file=sys.stderr)
    if failures:
        raise RuntimeError("nvcc failed:\n" + "\n".join(failures))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc, *ARCH, "-shared", "--cudart", "static", "-o", str(tmp), *map(str, objects), "-ldl"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("link failed:\n" + res.stdout + res.stderr)
    os.replace(tmp, LIB)
    build_binding(force, verbose)
    return LIB


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose=True))
