"""Ahead-of-time build of the sm_100a kernel library ``libmak_kvcache.so`` and of its Python entry ``_mak_front.so``.

The reference JIT-compiles its MUSA sources with ``mcc`` into a per-user cache
(musa_aiter/jit/core.py:31-95).  Here the CUDA sources under ``csrc/`` are
compiled once with ``nvcc -gencode arch=compute_100a,code=sm_100a`` into the
package's ``lib/`` folder, so the library travels with the source tree and no
GPU is needed to build it (nvcc cross-compiles).  ``csrc/front.cpp``, the
CPython module through which the short calls reach the library, is compiled
with the host compiler against the installed torch.
"""

from __future__ import annotations

import concurrent.futures
import hashlib
import importlib.metadata
import os
import shutil
import subprocess
import sys
import sysconfig
from dataclasses import dataclass
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
SOURCE_ROOT = PACKAGE_DIR.parent  # musa-aiter_b200/
REPO_ROOT = SOURCE_ROOT.parent
CSRC_DIR = SOURCE_ROOT / "csrc"
INCLUDE_DIR = REPO_ROOT / "include"
LIB_DIR = PACKAGE_DIR / "lib"
LIB_NAME = "libmak_kvcache.so"
LIB_PATH = LIB_DIR / LIB_NAME
FRONT_SOURCE = CSRC_DIR / "front.cpp"
FRONT_PATH = LIB_DIR / "_mak_front.so"
BUILD_DIR = SOURCE_ROOT / "_build"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC,-O3,-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


@dataclass(frozen=True)
class BuildResult:
    ok: bool
    message: str
    library_path: Path | None


def _nvcc() -> str | None:
    cand = os.environ.get("NVCC")
    if cand and Path(cand).exists():
        return cand
    found = shutil.which("nvcc")
    if found:
        return found
    default = Path("/usr/local/cuda/bin/nvcc")
    return str(default) if default.exists() else None


def sources() -> list[Path]:
    return sorted(CSRC_DIR.glob("*.cu"))


def _fingerprint(front: bool) -> str:
    """Of what the library, or the Python entry, is built from."""
    h = hashlib.sha256()
    headers = sorted(INCLUDE_DIR.glob("*.h"))
    for path in [FRONT_SOURCE] + headers if front else sources() + sorted(CSRC_DIR.glob("*.cuh")) + headers:
        h.update(path.name.encode())
        h.update(path.read_bytes())
    h.update(" ".join([importlib.metadata.version("torch"), sys.version] if front else ARCH_FLAGS + NVCC_FLAGS).encode())
    return h.hexdigest()


def _is_current(path: Path, front: bool) -> bool:
    stamp = _stamp_path(path)
    return path.exists() and stamp.exists() and stamp.read_text().strip() == _fingerprint(front)


def _stamp_path(path: Path) -> Path:
    return path.with_name(path.name + ".stamp")


def is_built() -> bool:
    return _is_current(LIB_PATH, False) and _is_current(FRONT_PATH, True)


def _front_command(out: Path) -> list[str]:
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc() or "/usr/local/cuda/bin/nvcc").resolve().parent.parent
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", str(INCLUDE_DIR),
            "-I", str(root / "include"), "-I", str(root / "include" / "torch" / "csrc" / "api" / "include"),
            "-I", str(cuda / "include"), "-I", sysconfig.get_paths()["include"], str(FRONT_SOURCE), "-o", str(out),
            "-L", str(root / "lib"), "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10", "-lc10_cuda"]


def build(force: bool = False, verbose: bool = False) -> BuildResult:
    """Compile every ``csrc/*.cu`` for sm_100a, link ``lib/libmak_kvcache.so`` and build ``lib/_mak_front.so``, each
    where its sources changed (the latter also for another torch or Python)."""
    with_lib, with_front = (force or not _is_current(path, front) for path, front in ((LIB_PATH, False), (FRONT_PATH, True)))
    if not with_lib and not with_front:
        return BuildResult(True, "up to date", LIB_PATH)
    nvcc = _nvcc()
    if with_lib and nvcc is None:
        return BuildResult(False, "nvcc compiler not found", None)
    BUILD_DIR.mkdir(parents=True, exist_ok=True)
    LIB_DIR.mkdir(parents=True, exist_ok=True)

    def run(cmd: list[str]) -> subprocess.CompletedProcess:
        if verbose:
            print(" ".join(cmd))
        return subprocess.run(cmd, capture_output=True, text=True)

    objects = [BUILD_DIR / (src.stem + ".o") for src in sources()] if with_lib else []
    front_tmp, lib_tmp = LIB_DIR / "_mak_front.so.tmp", LIB_DIR / (LIB_NAME + ".tmp")
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        jobs = [pool.submit(run, _front_command(front_tmp))] if with_front else []
        include = ["-I", str(INCLUDE_DIR), "-I", str(CSRC_DIR)]
        for src, obj in zip(sources() if with_lib else [], objects):
            jobs.append(pool.submit(run, [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, *include, "-c", str(src), "-o", str(obj)]))
        results = [job.result() for job in jobs]
    if with_lib and not any(proc.returncode for proc in results):
        results.append(run([nvcc, *ARCH_FLAGS, "-shared", "-o", str(lib_tmp), *map(str, objects)]))
    errors = [proc.stderr for proc in results if proc.returncode != 0]
    if errors:
        return BuildResult(False, "\n".join(errors), None)
    for tmp, path, front in ((lib_tmp, LIB_PATH, False), (front_tmp, FRONT_PATH, True)):
        if with_front if front else with_lib:
            os.replace(tmp, path)
            _stamp_path(path).write_text(_fingerprint(front) + "\n")
    return BuildResult(True, "built", LIB_PATH)


if __name__ == "__main__":  # pragma: no cover - manual entry point
    result = build(force=True, verbose=True)
    print(result.message)
    raise SystemExit(0 if result.ok else 1)
