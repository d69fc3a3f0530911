"""Build the sm_100a shared library ``computd_b200/libdwa_b200.so`` in-tree.

Usage: ``python -m computd_b200.build [--force] [--verbose]``.

Each ``csrc/*.cu`` is compiled with nvcc for ``sm_100a`` only (tcgen05/TMA
need the architecture-specific target) into ``computd_b200/_build/`` and
linked with a static CUDA runtime, so the library does not depend on the
runtime version torch ships.  ``csrc/host/serving.cpp``, the Python side of the
serving calls, becomes the extension module ``computd_b200/_serving.so`` (host
compiler, torch's headers).  Objects are rebuilt when a source or header is
newer than them, the extension also when torch or Python is another than it was
built for.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
BUILD_DIR = PKG_DIR / "_build"
LIB_PATH = PKG_DIR / "libdwa_b200.so"
HOST_SOURCE = CSRC / "host" / "serving.cpp"
HOST_PATH = PKG_DIR / "_serving.so"
INCLUDE_DIR = REPO_DIR / "include"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON_FLAGS = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=hidden",
    "-Xcompiler", "-Wall",
    f"-I{INCLUDE_DIR}",
]


def nvcc_path() -> str:
    cand = shutil.which("nvcc")
    if cand:
        return cand
    default = "/usr/local/cuda/bin/nvcc"
    if os.path.exists(default):
        return default
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build computd_b200")


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _headers() -> list[Path]:
    return sorted(list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE_DIR.glob("*.h")))


def _stale(obj: Path, deps: list[Path]) -> bool:
    if not obj.exists():
        return True
    t = obj.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _compile(nvcc: str, src: Path, obj: Path, verbose: bool, extra: list[str]) -> None:
    cmd = [nvcc, *ARCH_FLAGS, *COMMON_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}")


def _host_built_for() -> str:
    """What the extension module depends on beside its sources: the installed torch and Python."""
    import torch

    return f"{torch.__version__}\n{Path(torch.__file__).resolve().parent}\n{sys.version}\n"


def _host_note() -> Path:
    return BUILD_DIR / "serving_built_for.txt"


def _note_host() -> None:
    _host_note().write_text(_host_built_for())


def _host_stale() -> bool:
    note = _host_note()
    return (_stale(HOST_PATH, [HOST_SOURCE, *INCLUDE_DIR.glob("*.h"), Path(__file__)])
            or not note.exists() or note.read_text() != _host_built_for())


def _build_host(verbose: bool) -> None:
    """The extension module of the serving calls, against the installed torch and Python."""
    import sysconfig

    import torch

    torch_dir = Path(torch.__file__).resolve().parent
    cuda_inc = Path(nvcc_path()).resolve().parent.parent / "include"
    cxx = shutil.which("c++") or shutil.which("g++")
    if not cxx:
        raise RuntimeError("a C++ compiler is required to build computd_b200/_serving.so")
    tmp = HOST_PATH.with_suffix(".so.tmp")
    lib = torch_dir / "lib"
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE_DIR}",
           *(f"-isystem{p}" for p in (torch_dir / "include",
                                      torch_dir / "include/torch/csrc/api/include", cuda_inc,
                                      sysconfig.get_paths()["include"])),
           str(HOST_SOURCE), "-o", str(tmp), f"-L{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu",
           "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"{cxx} failed on {HOST_SOURCE.name}")
    os.replace(tmp, HOST_PATH)
    _note_host()


def build(force: bool = False, verbose: bool = False, extra_flags: list[str] | None = None) -> Path:
    """Compile and link the library and the serving extension; returns the library's path."""
    nvcc = nvcc_path()
    extra = list(extra_flags or [])
    BUILD_DIR.mkdir(exist_ok=True)
    headers = _headers()
    objs = []
    jobs = []
    for src in _sources():
        obj = BUILD_DIR / (src.stem + ".o")
        objs.append(obj)
        if force or _stale(obj, [src, *headers, Path(__file__)]):
            jobs.append((src, obj))
    host = force or _host_stale()
    if jobs or host:
        with cf.ThreadPoolExecutor(max_workers=min(len(jobs) + 1, os.cpu_count() or 4)) as ex:
            futs = [ex.submit(_compile, nvcc, s, o, verbose, extra) for s, o in jobs]
            if host:
                futs.append(ex.submit(_build_host, verbose))
            for f in futs:
                f.result()
    if force or jobs or _stale(LIB_PATH, objs):
        tmp = LIB_PATH.with_suffix(".so.tmp")
        cmd = [nvcc, *ARCH_FLAGS, "-shared", "-cudart", "static", "-o", str(tmp),
               *[str(o) for o in objs]]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("linking libdwa_b200.so failed")
        os.replace(tmp, LIB_PATH)
    return LIB_PATH


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true", help="nvcc command lines and -Xptxas -v")
    args = ap.parse_args(argv)
    path = build(force=args.force, verbose=args.verbose)
    print(path)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
