"""Build libqmla.so in-tree for sm_100a with nvcc.

    python -m qwen_mla_vllm_b200.build [--force]

The library is a plain shared object (static CUDA runtime, no libcuda link:
the TMA descriptor encoder is fetched at run time through the runtime's
driver entry-point query), so it loads on machines without a GPU driver and
its host-only entry points (qmla_plan, ...) work there.  Every ``csrc/*.cu``
is one object under ``build/``; the objects are compiled side by side, and
only those whose sources (from nvcc's dependency files) changed.
"""
from __future__ import annotations

import argparse
import os
import pathlib
import shlex
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

PKG = pathlib.Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OUT = PKG / "libqmla.so"
OBJ = ROOT / "build" / "qmla"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-diag-suppress", "177",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and pathlib.Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[pathlib.Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [ROOT / "include" / "qmla.h"]


def up_to_date() -> bool:
    if not OUT.exists():
        return False
    t = OUT.stat().st_mtime
    return all(s.stat().st_mtime <= t for s in sources())


def _object_current(src: pathlib.Path, obj: pathlib.Path) -> bool:
    """The object is newer than its source and every project header it was compiled from."""
    dep = obj.with_suffix(".d")
    if not obj.exists() or not dep.exists():
        return False
    t = obj.stat().st_mtime
    names = shlex.split(dep.read_text().replace("\\\n", " "))[1:]
    own = [pathlib.Path(n) for n in names if str(ROOT) in str(pathlib.Path(n).resolve())] + [src]
    return all(p.exists() and p.stat().st_mtime <= t for p in own)


def _compile(src: pathlib.Path, force: bool, verbose: bool) -> pathlib.Path:
    obj = OBJ / (src.stem + ".o")
    if not force and _object_current(src, obj):
        return obj
    cmd = [nvcc(), *NVCC_FLAGS, f"-I{ROOT / 'include'}", f"-I{CSRC}", "-MD", "-MF", str(obj.with_suffix(".d")),
           "-c", "-o", str(obj), str(src)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    return obj


def build(force: bool = False, verbose: bool = False) -> pathlib.Path:
    if not force and up_to_date():
        return OUT
    OBJ.mkdir(parents=True, exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    with ThreadPoolExecutor(len(srcs)) as pool:
        objs = list(pool.map(lambda s: _compile(s, force, verbose), srcs))
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [nvcc(), *NVCC_FLAGS[:2], "-shared", "-Xcompiler", "-fPIC", "-o", str(tmp), *map(str, objs)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    tmp.replace(OUT)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=True))
