"""CPU tests of the build's own rules: what it leaves behind where the torch side cannot be made, and when that is made again."""

import os
import sys

import pytest

from jax_linear_attention_b200 import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source tree of one small kernel file and a torch side of one line, in place of the real ones."""
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "one.cu").write_text('extern "C" int one() { return 1; }\n')
    (tmp_path / "csrc" / "torch_ops.cpp").write_text("int torch_side = 1;\n")
    for name, path in (("CSRC", "csrc"), ("OBJ", "build"), ("LIB", "lib.so"), ("TORCH_OPS", "_torch_ops.so")):
        monkeypatch.setattr(build, name, str(tmp_path / path))
    monkeypatch.setattr(build, "_torch_ops_command", lambda: ["g++", "-shared", "-fPIC", str(tmp_path / "csrc" / "torch_ops.cpp"), "-o",
                                                              str(tmp_path / "_torch_ops.so")])
    return tmp_path


def test_library_is_there_where_the_torch_side_fails(tree):
    (tree / "csrc" / "torch_ops.cpp").write_text("no C++ at all\n")
    with pytest.raises(RuntimeError, match="torch side"):
        build.build()
    assert (tree / "lib.so").exists() and not (tree / "_torch_ops.so").exists()


def test_host_without_torch(tree, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # an import of it raises
    find = build.importlib.util.find_spec
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build() == str(tree / "lib.so") and (tree / "lib.so").exists()
    assert not (tree / "_torch_ops.so").exists() and "no torch" in capsys.readouterr().err


def test_torch_side_is_made_again_for_another_torch(tree, monkeypatch):
    import torch

    def made():
        build.build()
        return os.stat(tree / "_torch_ops.so").st_mtime_ns

    first = made()
    assert made() == first
    monkeypatch.setattr(torch, "__version__", "0.0")
    second = made()
    assert second != first and made() == second
    monkeypatch.setattr(sys, "version", "another Python")
    third = made()
    assert third != second and made() == third
    command = build._torch_ops_command()
    monkeypatch.setattr(build, "_torch_ops_command", lambda: [command[0], "-g", *command[1:]])
    fourth = made()
    assert fourth != third and made() == fourth
