"""What `make` builds and when, with stand-ins for the compilers and for Python: the library needs no torch, and the module of torch tensors is built again when another torch comes."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

COMPILER = """#!/bin/sh
echo "$@" >> calls
while [ $# -gt 0 ]; do [ "$1" = -o ] && echo built > "$2"; shift; done
"""
# a Python with the torch that the file `torch` names, or without one
PYTHON = """#!/bin/sh
[ -s torch ] || exit 1
case "$2" in *include*sysconfig*|*sysconfig*include*) echo "-Iflags-of-$(cat torch)";; *) cat torch;; esac
"""


@pytest.fixture
def tree(tmp_path):
    shutil.copy(os.path.join(ROOT, "Makefile"), tmp_path)
    shutil.copytree(os.path.join(ROOT, "booster_b200", "csrc"), tmp_path / "booster_b200" / "csrc")
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    for name, text in (("cc", COMPILER), ("py", PYTHON)):
        (tmp_path / name).write_text(text)
        (tmp_path / name).chmod(0o755)

    def make(torch):
        """the calls of the compilers, one a line"""
        (tmp_path / "torch").write_text(torch)
        (tmp_path / "calls").write_text("")
        subprocess.run(["make", f"NVCC={tmp_path}/cc", f"CXX={tmp_path}/cc", f"PYTHON={tmp_path}/py"], cwd=tmp_path, check=True, capture_output=True, text=True)
        return (tmp_path / "calls").read_text().splitlines()

    make.at = tmp_path / "booster_b200"
    return make


def test_the_library_needs_no_torch(tree):
    calls = tree("")
    assert (tree.at / "libbooster_b200.so").exists() and not (tree.at / "_serve.so").exists()
    assert any("engine.cu" in c for c in calls) and not any("serve_torch" in c for c in calls)
    assert tree("") == []


def test_the_module_is_built_for_the_torch_that_is_there(tree):
    tree("")
    for torch in ("2.9.0-cpython-312", "2.11.0+cu128-cpython-312", "2.9.0-cpython-312"):
        (call,) = tree(torch)
        assert "serve_torch.cpp" in call and f"flags-of-{torch}" in call
        assert (tree.at / "_serve.so").exists()
        assert tree(torch) == []
