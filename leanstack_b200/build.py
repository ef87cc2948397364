"""Build libleanb200.so (nvcc, sm_100a) and the front end _torch_front.so (host C++) in-tree.

``python -m leanstack_b200.build [--force] [--verbose] [--profiling]`` compiles
every ``csrc/*.cu`` into ``leanstack_b200/_lib/libleanb200.so``.
``--profiling`` defines ``LEANB200_PROFILING``, which adds the measurement
hooks (per-CTA timestamp buffers, the NVLink ping-pong probe) to the library;
the default build has none of them.  The library links
the shared CUDA runtime (``libcudart.so.12``), so inside a PyTorch process it
binds to the runtime PyTorch already loaded and sees the same current device
and streams.  ``csrc/torch_front.cpp`` becomes ``_lib/_torch_front.so``, a Python
module on the installed PyTorch's headers that calls the library; without PyTorch
or Python's headers it is left out, with a note, and the library alone serves the
C ABI.  No GPU is needed to build.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
OUT_DIR = PKG / "_lib"
LIB = OUT_DIR / "libleanb200.so"
OBJ_DIR = PKG / "_build"
FRONT_SRC = CSRC / "torch_front.cpp"
FRONT = OUT_DIR / "_torch_front.so"
FRONT_STAMP = OUT_DIR / "front_torch.txt"  # the PyTorch version that the front end was built for

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O2",
              "--expt-relaxed-constexpr", "-cudart", "shared"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put /usr/local/cuda/bin on PATH")


def cuda_home() -> Path:
    return Path(nvcc_path()).resolve().parent.parent


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _deps() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


STAMP = OUT_DIR / "build_flags.txt"


def _compile(src: Path, verbose: bool, ptxas_verbose: bool, defines: list[str]) -> tuple[Path, str]:
    obj = OBJ_DIR / (src.stem + ".o")
    cmd = [nvcc_path(), *ARCH_FLAGS, *NVCC_FLAGS, *defines, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src),
           "-o", str(obj)]
    if ptxas_verbose:
        cmd += ["-Xptxas", "-v"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    return obj, res.stderr


def torch_version() -> str | None:
    """Version of the installed PyTorch, None without one (imported only if it has no package data)."""
    if importlib.util.find_spec("torch") is None:
        return None
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:  # a PyTorch that was not installed as a package
        import torch

        return torch.__version__


def front_lacks() -> str | None:
    """What the front end needs and this machine does not have, None if all is there."""
    if torch_version() is None:
        return "PyTorch"
    if not (Path(importlib.util.find_spec("torch").origin).parent / "lib" / "libc10_cuda.so").exists():
        return "PyTorch with CUDA"
    if not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return "Python's headers"
    return None


def needs_front() -> bool:
    if not FRONT.exists() or not FRONT_STAMP.exists() or FRONT_STAMP.read_text().strip() != torch_version():
        return True
    return any(p.stat().st_mtime > FRONT.stat().st_mtime for p in [FRONT_SRC, *INCLUDE.glob("*.h"), Path(__file__)])


def build_front(verbose: bool = False) -> Path | None:
    """Compile the front end against the installed PyTorch and link it to libleanb200.so beside it."""
    lacks = front_lacks()
    if lacks:
        print(f"{FRONT.name} is left out: no {lacks}; {LIB.name} serves the C ABI", file=sys.stderr)
        return None
    import torch

    home = Path(torch.__file__).parent
    tmp = FRONT.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", str(home / "include"),
           "-I", str(home / "include" / "torch" / "csrc" / "api" / "include"), "-I", str(cuda_home() / "include"),
           "-I", sysconfig.get_paths()["include"], "-I", str(INCLUDE), str(FRONT_SRC), "-o", str(tmp),
           "-L", str(home / "lib"), "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10",
           "-L", str(OUT_DIR), f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"the front end failed to build:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, FRONT)
    FRONT_STAMP.write_text(torch_version() + "\n")
    return FRONT


def needs_build(defines: list[str] | None = None) -> bool:
    if not LIB.exists():
        return True
    if not STAMP.exists() or STAMP.read_text().split() != (defines or []):
        return True
    lib_mtime = LIB.stat().st_mtime
    return any(p.stat().st_mtime > lib_mtime for p in [*sources(), *_deps(), Path(__file__)])


def build(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False, profiling: bool = False) -> Path:
    defines = ["-DLEANB200_PROFILING"] if profiling else []
    if not force and not needs_build(defines):
        if needs_front():
            build_front(verbose)
        return LIB
    OUT_DIR.mkdir(parents=True, exist_ok=True)
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    for stale in OBJ_DIR.glob("*.o"):  # objects of sources that no longer exist must not be linked
        if not (CSRC / (stale.stem + ".cu")).exists():
            stale.unlink()
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=min(len(srcs), os.cpu_count() or 4)) as ex:
        results = list(ex.map(lambda s: _compile(s, verbose, ptxas_verbose, defines), srcs))
    if ptxas_verbose:
        for _, log in results:
            if log.strip():
                print(log)
    tmp = LIB.with_suffix(".so.tmp")
    lib64 = cuda_home() / "lib64"
    cmd = [nvcc_path(), *ARCH_FLAGS, "-shared", "-cudart", "shared", "-o", str(tmp), *[str(o) for o, _ in results],
           "-L", str(lib64), "-Xlinker", f"-rpath,{lib64}"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    STAMP.write_text(" ".join(defines) + "\n")
    build_front(verbose)
    return LIB


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-verbose", action="store_true", help="print registers / spills per kernel")
    ap.add_argument("--profiling", action="store_true", help="add the measurement hooks (LEANB200_PROFILING)")
    args = ap.parse_args(argv)
    lib = build(force=args.force, verbose=args.verbose, ptxas_verbose=args.ptxas_verbose, profiling=args.profiling)
    print(lib)
    return 0


if __name__ == "__main__":
    sys.exit(main())
