"""Build the sm_100a shared library ``piper_kernels/_lib/libpiper_b200.so``.

Usage: ``python piper-kernels_b200/build.py [--force] [--verbose] [--library-only]``.

Each ``csrc/*.cu`` is one translation unit, compiled by nvcc for ``sm_100a``
only (side by side) and linked into one library with the C ABI of
``include/piper_b200.h``.  The CUDA runtime is linked statically and the
driver's tensor-map encoder is looked up at run time, so the library has no
dependency beyond the NVIDIA driver, and building it needs nvcc alone.

``csrc/decoding_binding.cpp`` becomes a Python extension module beside it,
which calls the decoding entry points on torch tensors and needs torch's own
headers and libraries.  It is built after the library, again when torch
changes, and not without torch (nor with ``--library-only``).
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
BINDING_TORCH = OUTPUT.parent / "decoding_binding.torch"  # the torch that it was built with
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler", "-fPIC",
]


def sources() -> list[Path]:
    """What the library is made of."""
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [INCLUDE / "piper_b200.h"]


def binding_sources() -> list[Path]:
    return [CSRC / "decoding_binding.cpp", INCLUDE / "piper_b200.h"]


def is_current(output: Path, inputs: list[Path]) -> bool:
    return output.exists() and output.stat().st_mtime >= max(p.stat().st_mtime for p in inputs)


def torch_version() -> str | None:
    """The torch that a binding built now belongs to; None where there is none."""
    try:
        import torch
    except ImportError:
        return None
    return f"{torch.__version__} {torch._C._GLIBCXX_USE_CXX11_ABI}"


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


def build_library(directory: Path, verbose: bool) -> None:
    common = ["nvcc", *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", *(["-Xptxas", "-v"] if verbose else [])]
    units = [(src, directory / f"{src.stem}.o") for src in sorted(CSRC.glob("*.cu"))]
    running = [subprocess.Popen([*common, "-c", "-o", str(obj), str(src)]) for src, obj in units]
    codes = [process.wait() for process in running]
    for process, code in zip(running, codes):
        if code != 0:
            raise subprocess.CalledProcessError(code, process.args)
    subprocess.run(["nvcc", *NVCC_FLAGS, "-shared", "-o", str(OUTPUT), *(str(obj) for _, obj in units)], check=True)


def build_binding(directory: Path, version: str) -> None:
    obj = directory / "decoding_binding.o"
    subprocess.run([*binding_flags(), "-c", "-o", str(obj), str(CSRC / "decoding_binding.cpp")], check=True)
    # The binding finds the library beside it, and torch's are loaded with torch.
    subprocess.run(
        ["g++", "-shared", "-o", str(BINDING), str(obj), f"-L{OUTPUT.parent}", "-lpiper_b200",
         "-Wl,-rpath,$ORIGIN", *binding_libraries()], check=True)
    BINDING_TORCH.write_text(version)


def build(force: bool = False, verbose: bool = False, library_only: bool = False) -> Path:
    OUTPUT.parent.mkdir(parents=True, exist_ok=True)
    with tempfile.TemporaryDirectory() as tmp:
        if force or not is_current(OUTPUT, sources()):
            build_library(Path(tmp), verbose)
        if library_only:
            return OUTPUT
        version = torch_version()
        if version is None:
            print("torch is not installed: built the library without the Python binding", file=sys.stderr)
        elif (force or not is_current(BINDING, binding_sources()) or not BINDING_TORCH.exists()
              or BINDING_TORCH.read_text() != version):
            build_binding(Path(tmp), version)
    return OUTPUT


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--verbose", action="store_true")
    parser.add_argument("--library-only", action="store_true", help="no Python binding (needs nvcc alone)")
    args = parser.parse_args()
    print(build(force=args.force, verbose=args.verbose, library_only=args.library_only), file=sys.stderr)
