"""Builds libquailb200.so, the sm_100a kernel library, in-tree.

Each ``csrc/*.cu`` compiles to an object with nvcc for ``sm_100a`` only,
and the objects link into ``quail_b200/libquailb200.so`` with the CUDA
runtime linked statically, so the library carries no dependency on the
runtime version torch bundles. ``csrc/torch_ops.cpp``, the generation
operators' torch calls over that library's C ABI, compiles with g++ to
``quail_b200/_torch_ops.so``. Run as ``python -m quail_b200.build``.
"""

import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
CSRC = PACKAGE / "csrc"
INCLUDE = PACKAGE.parent / "include"
LIBRARY = PACKAGE / "libquailb200.so"
TORCH_OPS = PACKAGE / "_torch_ops.so"
BUILD_DIR = PACKAGE.parent / "_build"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
                "-Xcompiler", "-fPIC", "-I", str(INCLUDE)]


def nvcc() -> str:
    """Path of nvcc: CUDA_HOME first, then PATH, then /usr/local/cuda."""
    home = os.environ.get("CUDA_HOME")
    if home and (Path(home) / "bin" / "nvcc").exists():
        return str(Path(home) / "bin" / "nvcc")
    found = shutil.which("nvcc")
    if found:
        return found
    return "/usr/local/cuda/bin/nvcc"


def sources() -> list:
    return sorted(CSRC.glob("*.cu"))


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(Path(d).stat().st_mtime > t for d in deps)


def _compile(src: Path, verbose_ptxas: bool) -> Path:
    obj = BUILD_DIR / (src.stem + ".o")
    headers = list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    if not _stale(obj, [src, *headers]) and not verbose_ptxas:
        return obj
    cmd = [nvcc(), *ARCH_FLAGS, *COMMON_FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose_ptxas:
        cmd += ["-Xptxas", "-v"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{proc.stdout}\n{proc.stderr}")
    if verbose_ptxas:
        sys.stderr.write(proc.stderr)
    return obj


def _torch_build() -> str:
    """The torch and Python that _torch_ops.so is compiled for."""
    import torch
    return (f"torch {torch.__version__}, C++11 ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, "
            f"{sysconfig.get_config_var('SOABI')}")


def _build_torch_ops(force: bool) -> Path:
    src = CSRC / "torch_ops.cpp"
    built_for, now = BUILD_DIR / "torch_ops.for", _torch_build()
    same = built_for.exists() and built_for.read_text() == now
    if not force and same and not _stale(TORCH_OPS, [src, *INCLUDE.glob("*.h")]):
        return TORCH_OPS
    import torch
    root = Path(torch.__file__).parent
    tmp = TORCH_OPS.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", str(root / "include"),
           "-I", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-I", sysconfig.get_paths()["include"],
           "-I", str(Path(nvcc()).resolve().parent.parent / "include"), str(src), "-o", str(tmp),
           "-L", str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}:\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, TORCH_OPS)
    built_for.write_text(now)
    return TORCH_OPS


def build(force: bool = False, verbose_ptxas: bool = False) -> Path:
    """Compile every kernel source, link the shared library and build the torch
    calls over it.

    Returns:
        The path of libquailb200.so.
    """
    BUILD_DIR.mkdir(exist_ok=True)
    srcs = sources()
    if force:
        for obj in BUILD_DIR.glob("*.o"):
            obj.unlink()
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as pool:
        torch_ops = pool.submit(_build_torch_ops, force)
        objs = list(pool.map(lambda s: _compile(s, verbose_ptxas), srcs))
        torch_ops.result()
    if force or _stale(LIBRARY, objs):
        tmp = LIBRARY.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH_FLAGS, "-shared", "-cudart", "static", "-o", str(tmp),
               *map(str, objs), "-lcuda" if False else "-ldl"]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"link failed:\n{proc.stdout}\n{proc.stderr}")
        os.replace(tmp, LIBRARY)
    return LIBRARY


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose_ptxas="-v" in sys.argv)
    print(path)
