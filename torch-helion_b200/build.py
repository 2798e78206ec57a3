"""Build ``lib/libth_b200.so`` (all CUDA kernels + the C ABI) for sm_100a,
and ``lib/th_decode_ops.so`` (the Python entry points of the decoding
operators, ``csrc/decode_ops.cpp``, against the installed torch).

    python torch-helion_b200/build.py [--force] [--verbose]

The library is compiled in-tree with nvcc from ``csrc/th_b200.cu`` (a unity
translation unit) so it travels with the repository snapshot.  Beside it,
``libth_b200.so.sha256`` records a SHA-256 digest of every source under
``csrc/`` and ``include/`` plus the nvcc flags it was built from.  It is
rebuilt whenever that digest differs from the current sources' (file
contents, not modification times), and the loader refuses a library whose
digest does not match, so a binary in the tree is provably built from the
sources beside it.
"""

from __future__ import annotations

import argparse
import hashlib
import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
LIB = HERE / "lib" / "libth_b200.so"
BINDING = LIB.with_name("th_decode_ops.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17", "--expt-relaxed-constexpr",
    "-shared", "-Xcompiler", "-fPIC",
]

CXX_FLAGS = ["-O2", "-std=c++17", "-shared", "-fPIC", "-Wall"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


SHA = LIB.with_name(LIB.name + ".sha256")


def source_digest() -> str:
    """SHA-256 over the sources (path and contents, sorted) and the compilers' flags."""
    h = hashlib.sha256()
    srcs = sorted(f for d, ext in ((CSRC, "*.cu"), (CSRC, "*.cuh"), (CSRC, "*.cpp"), (INCLUDE, "*.h")) for f in d.glob(ext))
    for f in srcs:
        h.update(f.name.encode() + b"\0" + f.read_bytes() + b"\0")
    h.update(" ".join(NVCC_FLAGS + CXX_FLAGS).encode())
    return h.hexdigest()


def built_digest() -> str | None:
    return SHA.read_text().strip() if SHA.exists() and LIB.exists() and BINDING.exists() else None


def _stale() -> bool:
    return built_digest() != source_digest()


def _binding_command(out: Path) -> list[str]:
    import sysconfig

    import torch

    root = Path(torch.__file__).parent
    cuda = Path(_nvcc()).resolve().parent.parent
    include = [root / "include", root / "include/torch/csrc/api/include", cuda / "include", sysconfig.get_paths()["include"]]
    return [os.environ.get("CXX", "g++"), *CXX_FLAGS, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(x for d in include for x in ("-isystem", str(d))), str(CSRC / "decode_ops.cpp"), "-o", str(out),
            "-L" + str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not _stale():
        return LIB
    LIB.parent.mkdir(parents=True, exist_ok=True)
    digest = source_digest()
    jobs = []
    for out, cmd in ((LIB, lambda tmp: [_nvcc(), *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-o", str(tmp),
                                        str(CSRC / "th_b200.cu")]), (BINDING, _binding_command)):
        tmp = out.with_suffix(".so.tmp")
        jobs.append((out, tmp, subprocess.Popen(cmd(tmp), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
    done = [(out, tmp, job, job.communicate()) for out, tmp, job in jobs]
    for out, _, job, text in done:
        if job.returncode != 0:
            sys.stderr.write("".join(text))
            raise RuntimeError(f"compiling {out.name} failed ({job.returncode})")
        if verbose:
            sys.stderr.write(text[1])
    for out, tmp, _, _ in done:
        tmp.replace(out)
    SHA.write_text(digest + "\n")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
