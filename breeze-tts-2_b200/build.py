"""Build libbreeze_b200.so (sm_100a) in-tree with nvcc.

    python breeze-tts-2_b200/build.py [--force] [--jobs N]

Compiles every csrc/*.cu as relocatable device code (``WHOLE``: as a whole
program) for ``-gencode arch=compute_100a,code=sm_100a`` and links them, with
the CUDA runtime linked statically, into breeze_b200/libbreeze_b200.so next to
the Python package that loads it. Objects go to _build/ (git-ignored). The
library depends on nothing from PyTorch; breeze_b200/_paged_bind.so, the Python
side of the paged operators (csrc/bind_paged.cpp, host code), is compiled
against Python's and torch's headers. Where that fails there is a warning and no
such file, and the operators are called from Python alone.
"""

from __future__ import annotations

import argparse
import importlib.util
import os
import runpy
import shutil
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
OUT = HERE / "breeze_b200" / "libbreeze_b200.so"
BIND_SRC, BIND_OUT = CSRC / "bind_paged.cpp", HERE / "breeze_b200" / "_paged_bind.so"
BUILD = HERE / "_build"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
# compiled as whole programs: relocatable code ignores register reallocation (setmaxnreg)
WHOLE = {"bq_paged_wide", "bq_paged8_wide"}
CFLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-rdc=true", "--expt-relaxed-constexpr",
          f"-I{INCLUDE}", f"-I{CSRC}"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _stale(obj: Path, src: Path) -> bool:
    if not obj.exists():
        return True
    deps = [src, *CSRC.glob("*.h"), *CSRC.glob("*.cuh"), INCLUDE / "breeze_b200.h"]
    return any(d.stat().st_mtime > obj.stat().st_mtime for d in deps)


def torch_version() -> str | None:
    """Version of the installed torch, read without importing it."""
    spec = importlib.util.find_spec("torch")
    return None if spec is None else str(runpy.run_path(str(Path(spec.origin).parent / "version.py"))["__version__"])


def _bind_for() -> str:
    """What the bindings fit: the versions they were compiled against."""
    return f"{torch_version()} {sysconfig.get_config_var('SOABI')}"


def _bind_stale() -> bool:
    made = BUILD / "bind_for.txt"
    return _stale(BIND_OUT, BIND_SRC) or not made.exists() or made.read_text() != _bind_for()


def build_bind() -> str | None:
    """The Python side of the paged operators, against the installed torch. What went wrong, if anything did."""
    BIND_OUT.unlink(missing_ok=True)  # an old one might not fit the library
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return "torch is not installed"
    torch = Path(spec.origin).parent
    cuda = Path(nvcc()).resolve().parents[1]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-I{sysconfig.get_paths()['include']}", f"-I{torch / 'include'}", f"-I{torch / 'include/torch/csrc/api/include'}",
           f"-I{cuda / 'include'}", f"-I{INCLUDE}", f'-DBREEZE_TORCH_VERSION="{torch_version()}"', str(BIND_SRC), "-o", str(BIND_OUT), f"-L{torch / 'lib'}",
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", f"-Wl,-rpath,{torch / 'lib'}"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        return str(e)
    if r.returncode != 0:
        BIND_OUT.unlink(missing_ok=True)
        return f"{cmd[0]} failed on {BIND_SRC.name}:\n{r.stdout}\n{r.stderr}"
    (BUILD / "bind_for.txt").write_text(_bind_for())
    return None


def build(force: bool = False, jobs: int | None = None, verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    objs = [BUILD / (s.stem + ".o") for s in srcs]
    todo = [(s, o) for s, o in zip(srcs, objs) if force or _stale(o, s)]

    def compile_one(so):
        s, o = so
        flags = [f for f in CFLAGS if f != "-rdc=true"] if s.stem in WHOLE else CFLAGS
        cmd = [nvcc(), *ARCH, *flags, "-c", str(s), "-o", str(o)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {s.name}:\n{r.stdout}\n{r.stderr}")
        return r.stderr

    with ThreadPoolExecutor(max_workers=jobs or min(8, os.cpu_count() or 1)) as ex:
        bind = ex.submit(build_bind) if force or _bind_stale() else None
        for log in ex.map(compile_one, todo):
            if verbose and log:
                print(log)
    if todo or force or not OUT.exists():
        cmd = [nvcc(), *ARCH, "-shared", "-rdc=true", "-Xcompiler", "-fPIC", "-cudart", "static",
               *map(str, objs), "-o", str(OUT)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    why = None if bind is None else bind.result()
    if why is not None:
        warnings.warn(f"no {BIND_OUT.name} (the paged operators' calls then cost a few microseconds more): {why}", stacklevel=2)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, jobs=a.jobs, verbose=a.verbose))
    sys.exit(0)
