"""Build the Kitty B200 CUDA libraries in-tree.

    python kitty-kv_b200/build.py            # -> kitty-kv_b200/kitty/libkitty_b200.so, libkitty_kv8.so

Compiles every ``csrc/*.cu`` for sm_100a only (no PTX for other targets) with
IEEE float32 division and square root (no --use_fast_math: the quantisers must
round exactly like the reference) and links one shared library exporting the
C ABI declared in ``include/kitty_b200.h``; ``csrc/kv8/*.cu`` (the 8-bit cache) make
a second one with the C ABI of ``include/kitty_kv8.h``, and ``csrc/kv8/kv8_torch.cpp`` the
Python module that calls it with torch tensors.  Objects go to ``_build/``.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from importlib import metadata
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent
REPO_ROOT = PKG_ROOT.parent
CSRC = PKG_ROOT / "csrc"
BUILD = PKG_ROOT / "_build"
LIB = PKG_ROOT / "kitty" / "libkitty_b200.so"
LIB_KV8 = PKG_ROOT / "kitty" / "libkitty_kv8.so"
KV8_TORCH = PKG_ROOT / "kitty" / "kernels" / "_kv8_torch.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-prec-div=true", "-prec-sqrt=true", "-ftz=false", "-I", str(REPO_ROOT / "include")]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put CUDA's bin directory on PATH")


def build(verbose: bool = False, extra: list | None = None) -> Path:
    headers = [*CSRC.glob("*.cuh"), REPO_ROOT / "include" / "kitty_b200.h"]
    _library(LIB, CSRC.glob("*.cu"), headers, [], verbose, extra)
    headers = [*(CSRC / "kv8").glob("*.cuh"), *(REPO_ROOT / "include").glob("*.h")]
    _library(LIB_KV8, (CSRC / "kv8").glob("*.cu"), headers, ["-Xcompiler", "-fvisibility=hidden"], verbose, extra)
    _torch_module(KV8_TORCH, CSRC / "kv8" / "kv8_torch.cpp", LIB_KV8, verbose)
    return LIB


def _library(lib: Path, sources, headers, flags: list, verbose: bool, extra: list | None) -> None:
    """Compile what is older than its source or the headers (sources side by side) and link."""
    BUILD.mkdir(exist_ok=True)
    newest_header = max(h.stat().st_mtime for h in headers)
    objs, cmds = [], []
    for src in sorted(sources):
        obj = BUILD / (src.stem + ".o")
        objs.append(obj)
        if obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, newest_header):
            continue
        cmds.append([nvcc(), *ARCH, *NVCC_FLAGS, *flags, *(extra or []), "-c", str(src), "-o", str(obj)])
        if verbose:
            print(" ".join(cmds[-1]), flush=True)
    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        for done in [pool.submit(subprocess.run, cmd, check=True) for cmd in cmds]:
            done.result()
    if (not lib.exists()) or any(o.stat().st_mtime > lib.stat().st_mtime for o in objs):
        tmp = lib.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-Xlinker", f"-soname={lib.name}", "-o", str(tmp),
               *map(str, objs)]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        os.replace(tmp, lib)


def _torch_built_for() -> str:
    """What a module built against torch's C++ interface holds for."""
    try:
        torch_version = metadata.version("torch")
    except metadata.PackageNotFoundError:
        import torch
        torch_version = torch.__version__
    return f"torch {torch_version}, python {sys.version}\n"


def _torch_module(module: Path, src: Path, lib: Path, verbose: bool) -> None:
    """The Python extension module: the host compiler, torch's headers and libraries.  Built again
    for another torch or Python too, whose C++ interface may differ."""
    header = REPO_ROOT / "include" / "kitty_kv8.h"
    note, built_for = BUILD / (module.stem + ".txt"), _torch_built_for()
    if (module.exists() and module.stat().st_mtime >= max(src.stat().st_mtime, header.stat().st_mtime)
            and note.exists() and note.read_text() == built_for):
        return
    import torch
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    tmp = module.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{d}" for d in (root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
                                      cuda / "include", sysconfig.get_paths()["include"])),
           str(src), "-o", str(tmp), str(lib), "-Wl,-rpath,$ORIGIN/..", f"-L{root / 'lib'}",
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-ltorch_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, module)
    note.write_text(built_for)


if __name__ == "__main__":
    build(verbose="-q" not in sys.argv, extra=[a for a in sys.argv[1:] if a != "-q"])
    print(LIB)
