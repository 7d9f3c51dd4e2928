"""Build recipe for ``libkoemi_b200.so``, the sm_100a kernel library.

Every ``csrc/*.cu`` translation unit is compiled by nvcc for
``-gencode arch=compute_100a,code=sm_100a`` into an object under ``_build/``
(skipped when the object is newer than its sources), and the objects are
linked into ``lib/libkoemi_b200.so`` with a static CUDA runtime, so the
library depends on nothing but the driver. nvcc cross-compiles without a GPU.

``csrc/binding/*.cpp`` are compiled by g++ against the installed torch into
``lib/libkoemi_b200_torch.so``: the dispatcher ops and autograd formulas of the
training operators, which open the kernel library at run time.

Run ``python -m koemi_5hom_b200.build`` (or call :func:`build`).
"""
from __future__ import annotations

import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
SOURCE_DIR = PACKAGE_DIR / "csrc"
INCLUDE_DIR = PACKAGE_DIR.parent / "include"
BUILD_DIR = PACKAGE_DIR.parent / "_build"
LIBRARY_PATH = PACKAGE_DIR / "lib" / "libkoemi_b200.so"
BINDING_DIR = SOURCE_DIR / "binding"
BINDING_PATH = PACKAGE_DIR / "lib" / "libkoemi_b200_torch.so"

ARCH_FLAGS = ("-gencode", "arch=compute_100a,code=sm_100a")
NVCC_FLAGS = (
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler",
    "-fPIC,-fvisibility=hidden",
    "-Xptxas",
    "-warn-spills",
)


def find_nvcc() -> str:
    candidates = [os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"]
    for candidate in candidates:
        if candidate and Path(candidate).is_file():
            return candidate
    raise RuntimeError("nvcc was not found; set NVCC or put the CUDA toolkit on PATH")


def _headers() -> list[Path]:
    return sorted(SOURCE_DIR.glob("*.cuh")) + sorted(INCLUDE_DIR.glob("*.h"))


def _compile(nvcc: str, source: Path, verbose: bool) -> Path:
    target = BUILD_DIR / (source.stem + ".o")
    newest_input = max(p.stat().st_mtime for p in [source, *_headers(), Path(__file__)])
    if target.exists() and target.stat().st_mtime >= newest_input:
        return target
    command = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, "-I", str(INCLUDE_DIR), "-c", str(source), "-o", str(target)]
    if verbose:
        print(" ".join(command), flush=True)
    result = subprocess.run(command, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(f"nvcc failed on {source.name}:\n{result.stdout}\n{result.stderr}")
    if verbose and (result.stdout or result.stderr):
        print(result.stdout + result.stderr, flush=True)
    return target


def build_binding(verbose: bool = False) -> Path:
    """Compile the torch binding (skipped when newer than its inputs and the torch it was built for)."""
    import torch

    compiler = os.environ.get("CXX") or shutil.which("g++")
    if not compiler:
        raise RuntimeError("g++ was not found; set CXX")
    root = Path(torch.__file__).resolve().parent
    cuda = Path(find_nvcc()).resolve().parent.parent
    newest_header = max(p.stat().st_mtime for p in
                        [*BINDING_DIR.glob("*.h"), *INCLUDE_DIR.glob("*.h"), Path(__file__), root / "version.py"])
    sources = sorted(BINDING_DIR.glob("*.cpp"))
    if BINDING_PATH.exists() and BINDING_PATH.stat().st_mtime >= max(newest_header, *(p.stat().st_mtime for p in sources)):
        return BINDING_PATH
    BINDING_PATH.parent.mkdir(parents=True, exist_ok=True)
    BUILD_DIR.mkdir(parents=True, exist_ok=True)

    def run(command: list[str], what: str) -> None:
        if verbose:
            print(" ".join(command), flush=True)
        result = subprocess.run(command, capture_output=True, text=True)
        if result.returncode != 0:
            raise RuntimeError(f"{what} failed:\n{result.stdout}\n{result.stderr}")

    def compile_one(source: Path) -> Path:
        target = BUILD_DIR / f"binding_{source.stem}.o"
        if not target.exists() or target.stat().st_mtime < max(newest_header, source.stat().st_mtime):
            run([compiler, "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
                 f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                 "-I", str(INCLUDE_DIR), "-isystem", str(root / "include"),
                 "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
                 "-isystem", str(cuda / "include"), "-isystem", sysconfig.get_path("include"),
                 "-c", str(source), "-o", str(target)], f"compiling {source.name}")
        return target

    with concurrent.futures.ThreadPoolExecutor(max_workers=len(sources)) as pool:
        objects = list(pool.map(compile_one, sources))
    temporary = BINDING_PATH.with_suffix(".so.tmp")
    run([compiler, "-shared", *map(str, objects), "-o", str(temporary),
         # torch's own C++ library: one linked in statically, as some compilers do by
         # themselves, crashes where both sides' streams meet
         "-l:libstdc++.so.6", "-L", str(root / "lib"), "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-ltorch_python", "-ldl"],
        "linking the torch binding")
    os.replace(temporary, BINDING_PATH)
    return BINDING_PATH


def build(verbose: bool = False, jobs: int | None = None) -> Path:
    """Compile every kernel translation unit and link the shared library, and compile the torch binding."""
    nvcc = find_nvcc()
    BUILD_DIR.mkdir(parents=True, exist_ok=True)
    LIBRARY_PATH.parent.mkdir(parents=True, exist_ok=True)
    sources = sorted(SOURCE_DIR.glob("*.cu"))
    if not sources:
        raise RuntimeError(f"no CUDA sources under {SOURCE_DIR}")
    workers = jobs or min(len(sources), os.cpu_count() or 4)
    with concurrent.futures.ThreadPoolExecutor(max_workers=workers) as pool:
        binding = pool.submit(build_binding, verbose)
        objects = list(pool.map(lambda s: _compile(nvcc, s, verbose), sources))
        binding.result()
    newest_object = max(o.stat().st_mtime for o in objects)
    if LIBRARY_PATH.exists() and LIBRARY_PATH.stat().st_mtime >= newest_object:
        return LIBRARY_PATH
    temporary = LIBRARY_PATH.with_suffix(".so.tmp")
    command = [nvcc, *ARCH_FLAGS, "-shared", "-cudart", "static", "-o", str(temporary),
               *map(str, objects)]
    if verbose:
        print(" ".join(command), flush=True)
    result = subprocess.run(command, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(f"linking libkoemi_b200.so failed:\n{result.stdout}\n{result.stderr}")
    os.replace(temporary, LIBRARY_PATH)
    return LIBRARY_PATH


def main(argv: list[str] | None = None) -> int:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("-v", "--verbose", action="store_true")
    parser.add_argument("-j", "--jobs", type=int, default=None)
    arguments = parser.parse_args(argv)
    path = build(verbose=arguments.verbose, jobs=arguments.jobs)
    print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main())
