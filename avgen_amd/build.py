"""Build ``libavattn.so`` (the C-ABI HIP library) in-tree with hipcc for gfx950,
and ``_direct_calls.so`` (the direct calls of some of its functions from torch).

Usage: ``python -m avgen_amd.build`` (or ``__graft_entry__.build()``).  Each
``csrc/*.hip`` is compiled to an object under ``avgen_amd/_build/`` in
parallel, then linked into ``avgen_amd/libavattn.so``.  Always recompiles.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
BUILD = PKG / "_build"
LIB = PKG / "libavattn.so"
CALLS = PKG / "_direct_calls.so"
ARCH = "gfx950"

# Packed-fp32 VALU forms stay disabled (plain scalar fp32 code only).
HIP_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]


def hipcc() -> str:
    """Return the hipcc executable (ROCm install or PATH)."""
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found: the avattn HIP library cannot be built")


def _compile(src: Path, extra: list[str]) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [hipcc(), *HIP_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass does not know the packed-fp32 feature name; drop that
    # one harmless warning line and surface everything else.
    noise = "is not a recognized feature for this target"
    msg = "\n".join(line for line in (proc.stdout + proc.stderr).splitlines() if noise not in line)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{msg}")
    if msg.strip():
        print(msg, file=sys.stderr)
    return obj


def _build_calls() -> None:
    """Host code against the installed torch, whose libraries are loaded when it is
    imported."""
    import torch

    home = Path(torch.__file__).parent
    include = home / "include"
    tmp = CALLS.with_suffix(".so.tmp")
    cmd = [hipcc(), "-x", "c++", "-O2", "-std=c++20", "-fPIC", "-fvisibility=hidden", "-shared", "-Wall",
           "-Wno-unused-function", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", f"-I{INCLUDE}",
           *(f"-isystem{d}" for d in (include, include / "torch/csrc/api/include", "/opt/rocm/include",
                                      sysconfig.get_paths()["include"])),
           str(CSRC / "direct_calls.cpp"), "-o", str(tmp), f"-L{home / 'lib'}",
           "-ltorch_python", "-ltorch_hip", "-ltorch_cpu", "-lc10_hip", "-lc10"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for direct_calls.cpp:\n{proc.stdout}{proc.stderr}")
    if proc.stderr.strip():
        print(proc.stderr, file=sys.stderr)
    os.replace(tmp, CALLS)


def build(verbose: bool = False, extra_flags: list[str] | None = None) -> Path:
    """Compile every kernel source and link the shared library; build the direct calls;
    return the library's path."""
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    extra = list(extra_flags or [])
    if verbose:
        extra += ["-Rpass-analysis=kernel-resource-usage"]
    with ThreadPoolExecutor(max_workers=min(8, len(sources))) as pool:
        calls = pool.submit(_build_calls)
        objs = list(pool.map(lambda s: _compile(s, extra), sources))
        calls.result()
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stdout}{proc.stderr}")
    # A kernel whose host-side launch stub was not emitted links fine but
    # fails at load time; refuse such a library here.
    nm = subprocess.run(["nm", "-D", "--undefined-only", str(tmp)], capture_output=True, text=True)
    missing = [line.split()[-1] for line in nm.stdout.splitlines() if "__device_stub__" in line]
    if missing:
        raise RuntimeError(f"link produced undefined kernel stubs (compiler host-pass issue): {missing[:4]}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    path = build(verbose="-v" in sys.argv)
    print(path)
