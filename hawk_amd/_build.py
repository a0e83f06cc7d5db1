"""Build step of hawk's gfx950 target: compile ``libhawk_core.so`` and ``_bind.so`` in-tree.

The library is the C-ABI launcher (``csrc/hawk_core.cpp``) plus the
hand-written team-stage kernels (``csrc/hawk_team.hip``, ``csrc/hawk_linalg.hip``) and training stages
(``csrc/hawk_recurrence.hip``, ``csrc/hawk_rows.hip``, ``csrc/hawk_dropout.hip``, ``csrc/hawk_norm.hip``,
``csrc/hawk_sample.hip``, ``csrc/hawk_linear.hip``), built by ``hipcc`` for gfx950 only, each file by a compiler of its own.  Beside it ``_bind.so`` (``csrc/hawk_bind.cpp``,
built by the host compiler against PyTorch's headers) checks and binds a stage's tensors; the library
is built and used without it.  The build digest is the sha256 of its own sources (each
file's name and sha256, in sorted order), stamped into both and
recomputed by :mod:`hawk_amd._core` at load, the same self-check the
reference runs at import (reference ``hawk/__init__.py:146-212``).
"""

from __future__ import annotations

import hashlib
import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
CSRC = PACKAGE / "csrc"
INCLUDE = ROOT / "include"
LIBRARY = PACKAGE / "libhawk_core.so"
BINDING = PACKAGE / "_bind.so"
HIPCC = os.environ.get("HAWK_HIPCC", "/opt/rocm/bin/hipcc")

#: The library's translation units.
UNITS = ("hawk_core.cpp", "hawk_team.hip", "hawk_linalg.hip", "hawk_recurrence.hip", "hawk_rows.hip",
         "hawk_dropout.hip", "hawk_norm.hip", "hawk_sample.hip", "hawk_linear.hip")

#: Flags every HIP translation unit of this target is built with: gfx950
#: only, no floating-point contraction (the host oracle's ``native`` profile
#: is built with -ffp-contract=off, reference hawk/compile/toolchain.py:956-987),
#: and packed-FP32 instruction selection switched off.
HIP_FLAGS = ("--offload-arch=gfx950", "-O3", "-ffp-contract=off",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops")


def digest_sources() -> list:
    """The files the build digest covers, relative to the repository root."""
    files = sorted(p for p in CSRC.iterdir() if p.is_file() and p.suffix in (".cpp", ".hip", ".h"))
    return files + [INCLUDE / "hawk_core.h"]


def source_digest() -> str:
    """sha256 over ``name\\nsha256(file)\\n`` of every covered file, sorted by name."""
    stream = []
    for path in sorted(digest_sources(), key=lambda p: p.relative_to(ROOT).as_posix()):
        stream.append(f"{path.relative_to(ROOT).as_posix()}\n{hashlib.sha256(path.read_bytes()).hexdigest()}\n")
    return hashlib.sha256("".join(stream).encode()).hexdigest()


def binding_command(digest: str, out: Path) -> list:
    """The host compiler's command for ``_bind.so``."""
    import sysconfig

    import torch
    at = Path(torch.__file__).resolve().parent
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f'-DHAWK_BUILD_DIGEST="{digest}"',
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{sysconfig.get_paths()['include']}",
            f"-I{at}/include", f"-I{at}/include/torch/csrc/api/include", str(CSRC / "hawk_bind.cpp"), "-o", str(out),
            f"-L{at}/lib", "-ltorch_python", "-ltorch_cpu", "-lc10"]


def _call(cmd: list, what: Path, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed building {what.name}:\n{proc.stdout}\n{proc.stderr}")


def build_library(verbose: bool = False) -> Path:
    """Compile ``libhawk_core.so`` next to this file; returns its path."""
    digest = source_digest()
    info = "compiler=" + HIPCC + "\\nflags=" + " ".join(HIP_FLAGS) + "\\noffload_arch=gfx950"
    tmp = LIBRARY.with_suffix(".so.tmp")
    flags = [*HIP_FLAGS, "-fPIC", "-std=c++17", f"-I{INCLUDE}", f"-I{CSRC}",
             f'-DHAWK_BUILD_DIGEST="{digest}"', f'-DHAWK_BUILD_INFO="{info}"']
    with tempfile.TemporaryDirectory() as made, ThreadPoolExecutor(len(UNITS)) as pool:
        objects = [str(Path(made) / f"{name}.o") for name in UNITS]
        list(pool.map(lambda pair: _call([HIPCC, *flags, "-c", str(CSRC / pair[0]), "-o", pair[1]], LIBRARY, verbose),
                      zip(UNITS, objects)))
        _call([HIPCC, "--offload-arch=gfx950", "-fPIC", "-shared", *objects, "-o", str(tmp), "-lhiprtc", "-lamdhip64"],
              LIBRARY, verbose)
    os.replace(tmp, LIBRARY)
    return LIBRARY


def build_binding(verbose: bool = False) -> Path:
    """Compile ``_bind.so`` next to this file (the training stages need it, nothing
    else does); returns its path."""
    tmp = BINDING.with_suffix(".so.tmp")
    _call(binding_command(source_digest(), tmp), BINDING, verbose)
    os.replace(tmp, BINDING)
    return BINDING


def build(verbose: bool = False) -> list:
    """Both, at the same time; returns their paths.  The library is in place where
    only the binding fails."""
    with ThreadPoolExecutor(1) as pool:
        binding = pool.submit(build_binding, verbose)
        return [build_library(verbose), binding.result()]


if __name__ == "__main__":
    print(*build(verbose="-v" in sys.argv), sep="\n")
