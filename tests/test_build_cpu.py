"""CPU: what build.py yields when a part of it cannot be built (the compilers are stand-ins)."""
import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """build.py with its outputs in tmp_path and an nvcc that writes an empty output file."""
    spec = importlib.util.spec_from_file_location("build_under_test", ROOT / "llm-decode-triton-6gb_b200" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    nvcc = tmp_path / "nvcc"
    nvcc.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do if [ "$1" = -o ]; then : > "$2"; fi; shift; done\n')
    nvcc.chmod(0o755)
    monkeypatch.setattr(mod, "nvcc_path", lambda: str(nvcc))
    monkeypatch.setattr(mod, "LIB_PATH", tmp_path / "libb200decode.so")
    monkeypatch.setattr(mod, "BINDING_PATH", tmp_path / "_binding.so")
    return mod


def failing(*args):
    return subprocess.CompletedProcess(args, 1, "", "no Python.h\n")


def test_a_binding_that_does_not_compile_leaves_the_library(builder, monkeypatch):
    monkeypatch.setattr(builder, "_build_binding", failing)
    with pytest.raises(RuntimeError, match="binding"):
        builder.build()
    assert builder.LIB_PATH.exists() and not builder.BINDING_PATH.exists()
    assert builder.needs_build()


def test_without_a_cpp_compiler_the_library_is_built(builder, monkeypatch):
    monkeypatch.setattr(builder.shutil, "which", lambda name: None)
    monkeypatch.setenv("PATH", "/bin/nowhere")
    monkeypatch.setattr(builder, "_compile", lambda src, obj, verbose: subprocess.run(["/bin/sh", builder.nvcc_path(), "-o", str(obj)], capture_output=True, text=True))
    with pytest.raises(RuntimeError, match="binding"):
        builder.build()
    assert builder.LIB_PATH.exists()


def test_the_library_alone(builder, monkeypatch):
    """A host without Python's torch: no binding is asked for or built."""
    monkeypatch.setitem(sys.modules, "torch", None)
    assert builder.build() == builder.LIB_PATH and builder.LIB_PATH.exists()
    assert not builder.BINDING_PATH.exists() and not builder.needs_build()
    monkeypatch.delitem(sys.modules, "torch")
    monkeypatch.setattr(builder, "_build_binding", failing)
    builder.build(force=True, binding=False)


def test_kernels_that_do_not_compile_fail_the_build(builder, monkeypatch):
    monkeypatch.setattr(builder, "_compile", failing)
    with pytest.raises(RuntimeError, match="compiler"):
        builder.build(binding=False)
    assert not builder.LIB_PATH.exists()


def test_a_binding_of_another_torch_is_rebuilt(builder):
    """The module calls torch's C++ ABI: one that was built against another torch or Python is out of date, however new
    the file is."""
    builder.LIB_PATH.write_bytes(b"")
    for built_for, needed in ((b"b2d built for " + builder.host_tag().encode() + b"\0", False), (b"b2d built for torch 1.0.0 cpython-312\0", True),
                              (b"", True)):
        builder.BINDING_PATH.write_bytes(b"\x7fELF" + built_for)
        assert builder.needs_build() is needed
    real = ROOT / "llm-decode-triton-6gb_b200" / "b200kernels" / "_binding.so"
    assert b"b2d built for " + builder.host_tag().encode() + b"\0" in real.read_bytes()


def test_a_binding_of_another_torch_is_not_used(monkeypatch):
    import torch
    from b200kernels import _lib
    monkeypatch.setattr(_lib, "_binding", None)
    assert _lib.binding() is not None
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    with pytest.raises(RuntimeError, match="built for torch .* not for torch 1.0.0"):
        _lib.binding()
    assert _lib._binding is None
