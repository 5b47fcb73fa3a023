"""Build the sm_100a shared library ``piper_kernels/_lib/libpiper_b200.so``.

Usage: ``python piper-kernels_b200/build.py [--force] [--verbose]``.

Each ``csrc/*.cu`` is one translation unit, compiled by nvcc for ``sm_100a``
only (side by side) and linked into one library with the C ABI of
``include/piper_b200.h``.  The CUDA runtime is linked statically and the
driver's tensor-map encoder is looked up at run time, so the library has no
dependency beyond the NVIDIA driver.  ``csrc/decoding_binding.cpp`` becomes a
Python extension module beside it, which calls the decoding entry points on
torch tensors and needs torch's own libraries.
"""

from __future__ import annotations

import argparse
import subprocess
import sys
import tempfile
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent
REPO_ROOT = PKG_ROOT.parent
CSRC = PKG_ROOT / "csrc"
INCLUDE = REPO_ROOT / "include"
OUTPUT = PKG_ROOT / "piper_kernels" / "_lib" / "libpiper_b200.so"
BINDING = OUTPUT.parent / "decoding_binding.so"
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler", "-fPIC",
]


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cpp")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [INCLUDE / "piper_b200.h"]


def binding_flags() -> list[str]:
    """The host compiler and its flags for ``csrc/decoding_binding.cpp`` (torch's C++ interface)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    includes = [*cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"]]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-w",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
            *(f"-I{path}" for path in includes)]


def binding_libraries() -> list[str]:
    from torch.utils import cpp_extension

    return [*(f"-L{path}" for path in cpp_extension.library_paths()), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
            "-ltorch_python"]


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and OUTPUT.exists() and BINDING.exists():
        newest = max(p.stat().st_mtime for p in sources())
        if min(OUTPUT.stat().st_mtime, BINDING.stat().st_mtime) >= newest:
            return OUTPUT
    OUTPUT.parent.mkdir(parents=True, exist_ok=True)
    common = ["nvcc", *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", *(["-Xptxas", "-v"] if verbose else [])]
    with tempfile.TemporaryDirectory() as tmp:
        units = [(src, Path(tmp) / f"{src.stem}.o") for src in sorted(CSRC.glob("*.cu"))]
        commands = [[*common, "-c", "-o", str(obj), str(src)] for src, obj in units]
        binding = Path(tmp) / "decoding_binding.o"
        commands.append([*binding_flags(), "-c", "-o", str(binding), str(CSRC / "decoding_binding.cpp")])
        running = [subprocess.Popen(command) for command in commands]
        codes = [process.wait() for process in running]
        for process, code in zip(running, codes):
            if code != 0:
                raise subprocess.CalledProcessError(code, process.args)
        subprocess.run(["nvcc", *NVCC_FLAGS, "-shared", "-o", str(OUTPUT), *(str(obj) for _, obj in units)], check=True)
        # The binding finds the library beside it, and torch's are loaded with torch.
        subprocess.run(
            ["g++", "-shared", "-o", str(BINDING), str(binding), f"-L{OUTPUT.parent}", "-lpiper_b200",
             "-Wl,-rpath,$ORIGIN", *binding_libraries()], check=True)
    return OUTPUT


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--verbose", action="store_true")
    args = parser.parse_args()
    print(build(force=args.force, verbose=args.verbose), file=sys.stderr)
