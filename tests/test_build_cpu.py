"""The library's build without the native calls' module (compilers that only write their output)."""
from __future__ import annotations

import warnings

import pytest

from conftest import dpa_mod

B = dpa_mod("build")


@pytest.fixture
def build(tmp_path, monkeypatch):
    cc = tmp_path / "cc"
    cc.write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\necho built > "$2"\n')
    cc.chmod(0o755)
    for name, path in (("BUILD_DIR", "_build"), ("LIB_DIR", "lib"), ("LIB_PATH", "lib/libdpa_fp8.so"),
                       ("FAST_PATH", "lib/dpa_fast_calls.so")):
        monkeypatch.setattr(B, name, tmp_path / path)
    monkeypatch.setattr(B, "hipcc", lambda: str(cc))
    monkeypatch.setattr(B, "_fast_calls_command",
                        lambda: [str(cc), "-o", str(B.FAST_PATH.with_suffix(".so.tmp"))])
    return tmp_path


def test_both_are_built(build):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert B.build_library() == B.LIB_PATH
    assert B.LIB_PATH.exists() and B.FAST_PATH.exists()


@pytest.mark.parametrize("kind", ["does not compile", "no torch", "no g++"])
def test_the_library_is_built_without_the_module(build, kind, monkeypatch):
    B.build_library()       # (what an earlier build left does not stay)

    def no_torch():
        raise ImportError("no torch here")
    command = {"does not compile": lambda: ["sh", "-c", "echo no such header; exit 1"], "no torch": no_torch,
               "no g++": lambda: [str(build / "none")]}[kind]
    monkeypatch.setattr(B, "_fast_calls_command", command)
    B.LIB_PATH.unlink()
    with pytest.warns(UserWarning, match="go through Python"):
        assert B.build_library() == B.LIB_PATH
    assert B.LIB_PATH.exists() and not B.FAST_PATH.exists()


def test_a_kernel_that_does_not_compile_fails_the_build(build, monkeypatch):
    cc = build / "bad"
    cc.write_text("#!/bin/sh\necho broken\nexit 1\n")
    cc.chmod(0o755)
    monkeypatch.setattr(B, "hipcc", lambda: str(cc))
    with pytest.raises(RuntimeError, match="broken"):
        B.build_library()
