"""Build libb200decode.so (all CUDA kernels + the C ABI) in-tree for sm_100a.

    python llm-decode-triton-6gb_b200/build.py [--verbose] [--force] [--no-binding]

The shared library lands next to the Python package (``b200kernels/libb200decode.so``) so it
travels with the source tree; nothing is installed into site-packages. The CPython module of the paged-cache and
draft-verification calls (``b200kernels/_binding.so``) is built beside it where torch is installed; hosts that use the
C ABI alone need neither it nor torch (``--no-binding``).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent
REPO_ROOT = PKG_ROOT.parent
CSRC = PKG_ROOT / "csrc"
INCLUDE = REPO_ROOT / "include"
LIB_PATH = PKG_ROOT / "b200kernels" / "libb200decode.so"
BINDING_PATH = PKG_ROOT / "b200kernels" / "_binding.so"   # CPython module of csrc/binding.cpp
SOURCES = ["capi.cu", "nf4_gemm.cu", "nf4_gemm_tma.cu", "nf4_tc5.cu", "nf4_format.cu", "gqa_decode.cu", "decode_glue.cu", "tp_allreduce.cu", "lm_head.cu",
           "paged_append.cu", "paged_attention.cu", "paged_prefix.cu", "verify_drafts.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libb200decode.so")
    return cand


def _older(path: Path, deps) -> bool:
    return not path.exists() or any(p.stat().st_mtime > path.stat().st_mtime for p in deps if p.exists())


def needs_library() -> bool:
    return _older(LIB_PATH, [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + [INCLUDE / "b200decode.h", Path(__file__)])


def _has_torch() -> bool:
    try:
        import torch  # noqa: F401
    except ImportError:
        return False
    return True


def host_tag() -> str:
    """What the binding depends on (``b200kernels/_lib.py`` compares the same text when it loads the module)."""
    import torch
    return f"torch {torch.__version__} {sys.implementation.cache_tag}"


def needs_binding() -> bool:
    if not _has_torch():
        return False
    return (_older(BINDING_PATH, [CSRC / "binding.cpp", INCLUDE / "b200decode.h", Path(__file__)])
            or f"b2d built for {host_tag()}\0".encode() not in BINDING_PATH.read_bytes())


def needs_build() -> bool:
    return needs_library() or needs_binding()


def _compile(src: Path, obj: Path, verbose: bool) -> subprocess.CompletedProcess:
    cmd = [nvcc_path(), "-c", "-Xcompiler", "-fPIC", "-O3", "-std=c++17", *ARCH, "-lineinfo", f"-I{INCLUDE}",
           "-o", str(obj), str(src)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd))
    return subprocess.run(cmd, capture_output=True, text=True)


def _build_binding(out: Path, verbose: bool) -> subprocess.CompletedProcess:
    """The CPython module against this interpreter's torch (its libraries are loaded by `import torch`)."""
    import sysconfig

    import torch
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parent.parent
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DB2D_HOST_TAG="{host_tag()}"',
           f"-I{INCLUDE}", f"-I{root / 'include'}", f"-I{root / 'include/torch/csrc/api/include'}", f"-I{cuda / 'include'}",
           f"-I{sysconfig.get_paths()['include']}", "-o", str(out), str(CSRC / "binding.cpp"),
           f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
           f"-Wl,-rpath,{root / 'lib'}"]
    if verbose:
        print(" ".join(cmd))
    return subprocess.run(cmd, capture_output=True, text=True)


def _report(res: subprocess.CompletedProcess, verbose: bool) -> bool:
    if verbose or res.returncode != 0:
        sys.stdout.write(res.stdout)
        sys.stderr.write(res.stderr)
    return res.returncode == 0


def _build_library(tmp: Path, verbose: bool) -> None:
    from concurrent.futures import ThreadPoolExecutor
    objs = [tmp / (Path(s).stem + ".o") for s in SOURCES]
    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 1)) as ex:
        results = list(ex.map(lambda so: _compile(CSRC / so[0], so[1], verbose), zip(SOURCES, objs)))
    if not all([_report(res, verbose) for res in results]):
        raise RuntimeError("the compiler failed")
    cmd = [nvcc_path(), "-shared", *ARCH, "-cudart", "shared", "-o", str(LIB_PATH) + ".tmp", *map(str, objs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if not _report(res, verbose):
        raise RuntimeError(f"nvcc link failed with exit code {res.returncode}")
    os.replace(str(LIB_PATH) + ".tmp", LIB_PATH)


def build(verbose: bool = False, force: bool = False, binding: bool = True) -> Path:
    """Compiles every source to an object file in parallel (one nvcc per source), then links the
    shared library; objects live in a temporary directory next to the library. The binding is compiled at the same
    time (not without torch, or with ``binding=False``); if it fails, that is raised once the library is in place."""
    import tempfile
    from concurrent.futures import ThreadPoolExecutor
    library = force or needs_library()
    with tempfile.TemporaryDirectory(dir=LIB_PATH.parent) as tmp, ThreadPoolExecutor(max_workers=1) as ex:
        made = None
        if binding and (_has_torch() if force else needs_binding()):
            made = ex.submit(_build_binding, Path(tmp) / BINDING_PATH.name, verbose)
        if library:
            _build_library(Path(tmp), verbose)
        if made is not None:
            try:
                ok = _report(made.result(), verbose)
            except OSError as e:   # no compiler
                raise RuntimeError(f"{BINDING_PATH.name}, the Python binding, could not be built: {e}") from e
            if not ok:
                raise RuntimeError(f"{BINDING_PATH.name}, the Python binding, does not compile")
            os.replace(Path(tmp) / BINDING_PATH.name, BINDING_PATH)
    return LIB_PATH


if __name__ == "__main__":
    build(verbose="--verbose" in sys.argv, force="--force" in sys.argv, binding="--no-binding" not in sys.argv)
    print(LIB_PATH)
