"""Build the lnet_b200 CUDA library in-tree for sm_100a.

``build()`` compiles every ``csrc/*.cu`` with nvcc into
``lnet_b200/_lib/liblnet_b200.so`` (a C-ABI shared library loaded with
ctypes), and ``csrc/torch_ops.cpp`` (the host path of the feed-forward and
distillation operators) with g++ against torch's headers into
``lnet_b200/_lib/_torch_ops.so``.  Rebuilds the library where a source or header
is newer, and the module where its sources, torch or Python are others than the
ones it was built from (``_torch_ops.stamp``): it shares structures with the
library and with torch, and another's must not be loaded.
"""

from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent  # the package directory holding csrc/
REPO = ROOT.parent
CSRC = ROOT / "csrc"
INCLUDE = REPO / "include"
LIB_DIR = PKG / "_lib"
LIB = LIB_DIR / "liblnet_b200.so"
TORCH_OPS_SOURCE = CSRC / "torch_ops.cpp"
TORCH_OPS = LIB_DIR / "_torch_ops.so"
ARCH = "-gencode=arch=compute_100a,code=sm_100a"


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; the lnet_b200 CUDA library cannot be built")
    return cand


def _sources():
    return sorted(CSRC.glob("*.cu"))


def _deps():
    return _sources() + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def needs_build() -> bool:
    if not LIB.exists():
        return True
    mtime = LIB.stat().st_mtime
    return any(p.stat().st_mtime > mtime for p in _deps())


def _torch_ops_stamp() -> str:
    """What the module is built from: its sources' text, torch and Python."""
    import torch

    h = hashlib.sha256(f"{torch.__version__} {sysconfig.get_config_var('SOABI')}".encode())
    for p in (TORCH_OPS_SOURCE, *sorted(INCLUDE.glob("*.h"))):
        h.update(p.read_bytes())
    return h.hexdigest()


def _stamp_path() -> Path:
    return TORCH_OPS.with_suffix(".stamp")


def torch_ops_stale() -> bool:
    if not TORCH_OPS.exists() or not _stamp_path().exists():
        return True
    return _stamp_path().read_text() != _torch_ops_stamp()


def _torch_ops_command(out: Path) -> list[str]:
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parents[1]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
            f"-I{root / 'include'}", f"-I{root / 'include/torch/csrc/api/include'}",
            f"-I{cuda / 'include'}", f"-I{sysconfig.get_paths()['include']}",
            str(TORCH_OPS_SOURCE), "-o", str(out), f"-L{root / 'lib'}", "-ltorch", "-ltorch_cpu",
            "-ltorch_python", "-lc10", "-lc10_cuda"]


def build_torch_ops(force: bool = False, verbose: bool = False) -> Path:
    if not force and not torch_ops_stale():
        return TORCH_OPS
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = TORCH_OPS.with_suffix(f".so.{os.getpid()}.tmp")
    stamp = _torch_ops_stamp()
    cmd = _torch_ops_command(tmp)
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed: {' '.join(cmd)}\n{res.stdout}{res.stderr}")
    _stamp_path().unlink(missing_ok=True)  # between the two the module counts as stale
    os.replace(tmp, TORCH_OPS)
    _stamp_path().write_text(stamp)
    return TORCH_OPS


def build(force: bool = False, verbose: bool = False) -> Path:
    """The library, which needs no torch, then the module."""
    build_library(force, verbose)
    build_torch_ops(force, verbose)
    return LIB


def build_library(force: bool = False, verbose: bool = False) -> Path:
    if not force and not needs_build():
        return LIB
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    obj_dir = ROOT / "_build"
    obj_dir.mkdir(exist_ok=True)
    nvcc = nvcc_path()
    flags = [
        "-O3", "-std=c++17", ARCH, "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
        f"-I{INCLUDE}", f"-I{CSRC}",
    ]
    objs = []
    procs = []
    for src in _sources():
        obj = obj_dir / (src.stem + ".o")
        objs.append(obj)
        cmd = [nvcc, *flags, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd))
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    for cmd, proc in procs:
        out, _ = proc.communicate()
        if proc.returncode != 0:
            raise RuntimeError(f"nvcc failed: {' '.join(cmd)}\n{out.decode()}")
        if verbose and out:
            print(out.decode())
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc, ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-lcublas"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed: {' '.join(cmd)}\n{res.stdout}{res.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    import sys

    print(build(force="--force" in sys.argv, verbose=True))
