"""In-tree build of libb2msl.so (the C-ABI kernel library) for sm_100a.

Every ``csrc/*.cu`` is compiled separately with nvcc (in parallel, only when
the source or a header changed) and linked into ``triton_msl_b200/libb2msl.so``
with the CUDA runtime linked statically, so the library carries no dependency
on the toolkit's shared cudart and travels with the source tree.
``csrc/binding.cpp``, the native Python binding of the decoder-serving operators,
is compiled against torch's headers into ``triton_msl_b200/_decoder.<python>.<torch>.so``:
its name holds the versions that its ABI goes by, so that another torch or Python builds
its own. One build runs at a time, whatever threads and processes ask for it.
"""
from __future__ import annotations

import concurrent.futures as cf
import contextlib
import fcntl
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libb2msl.so"
BINDING_SRC = CSRC / "binding.cpp"
INCLUDE = ROOT / "include"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH_FLAGS + [
    "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-Xptxas", "-warn-spills",
    "-I", str(INCLUDE),
]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; the kernel library cannot be built")
    return cand


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def _stale(obj: Path, src: Path, hdr_mtime: float) -> bool:
    if not obj.exists():
        return True
    m = obj.stat().st_mtime
    return m < src.stat().st_mtime or m < hdr_mtime


def _compile(src: Path, obj: Path, verbose: bool) -> tuple[Path, str]:
    cmd = [nvcc(), *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return src, r.stdout + r.stderr


def binding_path() -> Path:
    """The native binding for this Python and this torch."""
    import torch
    return PKG / f"_decoder.{sysconfig.get_config_var('SOABI')}.torch-{torch.__version__}.so"


@contextlib.contextmanager
def _alone():
    """Waits until no other thread or process builds."""
    BUILD.mkdir(exist_ok=True)
    with open(BUILD / ".lock", "w") as f:
        fcntl.flock(f, fcntl.LOCK_EX)
        yield


def _build_binding(force: bool) -> None:
    """Compile the native binding if its source or the C header changed."""
    binding = binding_path()
    newest = max(p.stat().st_mtime for p in (BINDING_SRC, *INCLUDE.glob("*.h")))
    if binding.exists() and not force and binding.stat().st_mtime >= newest:
        return
    import torch
    gxx = shutil.which("g++")
    if gxx is None:
        raise RuntimeError("g++ not found; the native binding cannot be built")
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    tmp = binding.with_name(binding.name + ".tmp")
    cmd = [gxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", str(root / "include"), "-I", str(root / "include/torch/csrc/api/include"),
           "-I", sysconfig.get_paths()["include"], "-I", str(cuda / "include"), str(BINDING_SRC), "-o", str(tmp),
           "-L", str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {BINDING_SRC.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, binding)


def build(force: bool = False, verbose: bool = False, jobs: int | None = None) -> Path:
    """Compile and link libb2msl.so and the native binding if anything changed. Returns
    the library's path."""
    with _alone():
        _build(force, verbose, jobs)
    return LIB


def _build(force: bool, verbose: bool, jobs: int | None) -> None:
    srcs = sorted(CSRC.glob("*.cu"))
    hdr_mtime = max((h.stat().st_mtime for h in _headers()), default=0.0)
    todo = []
    objs = []
    for s in srcs:
        o = BUILD / (s.stem + ".o")
        objs.append(o)
        if force or _stale(o, s, hdr_mtime):
            todo.append((s, o))
    logs = {}
    if todo:
        with cf.ThreadPoolExecutor(max_workers=jobs or min(len(todo), os.cpu_count() or 4)) as ex:
            for src, log in ex.map(lambda t: _compile(t[0], t[1], verbose), todo):
                logs[src.name] = log
    if todo or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH_FLAGS, "-shared", "-cudart", "static", "-o", str(tmp),
               *map(str, objs)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    if verbose:
        for name, log in sorted(logs.items()):
            print(f"== {name}\n{log}", file=sys.stderr)
    _build_binding(force)


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
