"""The build script, with the compilers replaced by scripts that leave files behind."""

import os

import pytest

from chronoquant_mlx_b200 import build as B


@pytest.fixture
def fake(tmp_path, monkeypatch):
    nvcc = tmp_path / "nvcc"
    nvcc.write_text('#!/bin/sh\nwhile [ "$1" != "-o" ]; do shift; done\necho built > "$2"\n')
    nvcc.chmod(0o755)
    src = tmp_path / "csrc"
    src.mkdir()
    for name in ("a", "b"):
        (src / f"{name}.cu").write_text("// a source\n")
    for name, value in dict(CSRC=str(src), OUT=str(tmp_path / "lib.so"), BUILD=str(tmp_path / "_build")).items():
        monkeypatch.setattr(B, name, value)
    monkeypatch.setattr(B, "nvcc", lambda: str(nvcc))
    return tmp_path


def test_the_library_is_linked_before_a_failing_extension_is_reported(fake, monkeypatch):
    """Bindings of the C ABI need the library alone: a g++ or torch headers that
    do not compile the extension leave it built."""
    def fails(force=False):
        raise RuntimeError("g++ failed")

    monkeypatch.setattr(B, "build_calls", fails)
    with pytest.raises(RuntimeError, match="g.. failed"):
        B.build()
    assert (fake / "lib.so").read_text() == "built\n"


def test_build_returns_the_library(fake, monkeypatch):
    monkeypatch.setattr(B, "build_calls", lambda force=False: "calls.so")
    assert B.build() == str(fake / "lib.so") and os.path.exists(fake / "_build" / "a.o")
