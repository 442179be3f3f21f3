"""Builds libenc_b200.so (the sm_100a kernel library) in-tree with nvcc.

    python -m enceladus_b200.build [--force] [--verbose]

Each .cu file under csrc/ is compiled to an object (in parallel) and linked into
enceladus_b200/lib/libenc_b200.so.  Objects are rebuilt when a source or header is newer.
csrc/torch_lane.cpp, the short way from torch tensors to the decoding step's entry points, becomes
enceladus_b200/lib/enc_torch_lane.so (host code only, g++ against torch's and Python's headers).  The library and
its binding work without it, so a host without those headers gets a message instead of an error.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

ROOT = Path(__file__).resolve().parent
CSRC = ROOT / "csrc"
LIBDIR = ROOT / "lib"
LIB = LIBDIR / "libenc_b200.so"
LANE = LIBDIR / "enc_torch_lane.so"
OBJDIR = ROOT / "build"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the kernel library cannot be built")
    return exe


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def needs_build() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + [ROOT.parent / "include" / "enceladus_b200.h"]
    return any(p.stat().st_mtime > t for p in deps)


def build_lane(force: bool = False, verbose: bool = False) -> Path | None:
    """Builds the torch lane where it is older than its sources; None where that is not possible."""
    import sysconfig
    from importlib.util import find_spec

    src = CSRC / "torch_lane.cpp"
    newest = max(p.stat().st_mtime for p in (src, ROOT.parent / "include" / "enceladus_b200.h"))
    if not force and LANE.exists() and LANE.stat().st_mtime >= newest:
        return LANE
    spec, cxx = find_spec("torch"), shutil.which("g++")
    python_h = Path(sysconfig.get_paths()["include"])
    try:
        cuda = Path(nvcc()).resolve().parents[1]
    except RuntimeError:
        cuda = None
    if spec is None or cxx is None or cuda is None or not (python_h / "Python.h").exists():
        sys.stderr.write("enc_torch_lane.so is not built (it needs g++, the CUDA toolkit, torch and Python's headers); calls go the longer way\n")
        return None
    torch = Path(spec.origin).parent
    LIBDIR.mkdir(exist_ok=True)
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", f"-I{torch}/include", f"-I{torch}/include/torch/csrc/api/include",
           f"-I{cuda}/include", f"-I{python_h}", str(src), "-o", str(LANE), f"-L{torch}/lib", "-ltorch_python", "-ltorch", "-ltorch_cpu",
           "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
    if r.returncode != 0:
        LANE.unlink(missing_ok=True)  # none rather than a stale one
        sys.stderr.write("enc_torch_lane.so could not be built; calls go the longer way\n")
        return None
    return LANE


def build(force: bool = False, verbose: bool = False) -> Path:
    build_lane(force, verbose)
    if not force and not needs_build():
        return LIB
    OBJDIR.mkdir(exist_ok=True)
    LIBDIR.mkdir(exist_ok=True)
    headers = list(CSRC.glob("*.cuh")) + [ROOT.parent / "include" / "enceladus_b200.h"]
    hdr_time = max(p.stat().st_mtime for p in headers)
    extra = ["-Xptxas", "-v"] if verbose else []

    def compile_one(src: Path) -> Path:
        obj = OBJDIR / (src.stem + ".o")
        if force or not obj.exists() or obj.stat().st_mtime < max(src.stat().st_mtime, hdr_time):
            cmd = [nvcc(), *NVCC_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
            r = subprocess.run(cmd, capture_output=True, text=True)
            if verbose or r.returncode != 0:
                sys.stderr.write(r.stdout + r.stderr)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src.name}")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objs = list(pool.map(compile_one, sources()))
    cmd = [nvcc(), "-shared", "-o", str(LIB), *map(str, objs), "-gencode", "arch=compute_100a,code=sm_100a"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("linking libenc_b200.so failed")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
