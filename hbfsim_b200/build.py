"""Build the in-tree CUDA library hbfsim_b200/libhbfsim_b200.so for sm_100a.

nvcc compiles the kernels and the C ABI directly (no torch extension
machinery): the library exports only extern "C" symbols with plain pointers,
so it can be bound from ctypes, cgo, JNI or a C/C++ host alike.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB = PKG / "libhbfsim_b200.so"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
SOURCES = ["timing.cu", "empirical.cu", "context.cu", "thermal.cu", "capacity.cu",
           "retention.cu", "prefetch.cu", "link.cu", "kv_append.cu", "kv_select.cu",
           "kv_attention.cu", "kv_evict.cu", "profile.cpp"]


def sources() -> list[Path]:
    return [CSRC / s for s in SOURCES]


def stale() -> bool:
    if not LIB.exists():
        return True
    built = LIB.stat().st_mtime
    deps = list(CSRC.glob("*")) + list((PKG.parent / "include" / "hbfsim").glob("*.h"))
    return any(p.stat().st_mtime > built for p in deps)


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc build of libhbfsim_b200.so failed")


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not stale():
        return LIB
    flags = [NVCC, *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC"]
    # exported C ABI: visibility comes from the version script below
    script = CSRC / "exports.map"
    with tempfile.TemporaryDirectory() as tmp:
        objects = [Path(tmp) / (src.stem + ".o") for src in sources()]
        with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:  # file by file
            list(pool.map(lambda x: _run([*flags, "-Xptxas", "-warn-spills", "-c", str(x[0]), "-o",
                                          str(x[1])], verbose), zip(sources(), objects)))
        made = Path(tmp) / LIB.name
        _run([*flags, "-shared", "-cudart", "static", "-o", str(made), *map(str, objects),
              "-Xlinker", f"--version-script={script}"], verbose)
        # in place at once: a process that has the old file loaded keeps it; under a name of its
        # own first: two builds at once do not write one file
        handle, staged = tempfile.mkstemp(prefix="." + LIB.stem + ".", suffix=".so", dir=LIB.parent)
        os.close(handle)
        try:
            shutil.copyfile(made, staged)
            os.chmod(staged, 0o755)
            os.replace(staged, LIB)
        except BaseException:
            os.unlink(staged)
            raise
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
