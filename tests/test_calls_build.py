"""The extension that shortens the way from Python to the library: what it is built for, and when (stand-ins for the compilers)."""

from __future__ import annotations

import shutil
import subprocess
import sys
import types

import pytest
import torch

from conftest import ROOT

import fast_dllm_relax_amd.vm as vm

PKG = ROOT / "fast-dllm-relax_amd"


def test_only_an_extension_for_this_torch_and_python_is_called():
    here = dict(torch=f"{torch.__version__} {torch.version.git_version}", python=sys.hexversion)
    assert vm.built_for_this(types.SimpleNamespace(**here))
    for other in (dict(here, torch="2.0.0 0000"), dict(here, torch=torch.__version__), dict(here, python=sys.hexversion + (1 << 16)), {},
                  dict(torch=here["torch"])):
        assert not vm.built_for_this(types.SimpleNamespace(**other))
    assert not vm.built_for_this(None)
    assert vm.fdllm_calls is None or vm.built_for_this(vm.fdllm_calls)


class Tree:
    """A copy of what the build reads, with stand-ins for the compilers and for Python that leave a line in `log`."""

    def __init__(self, tmp):
        self.pkg, self.log, self.tmp = tmp / "package", tmp / "log", tmp
        shutil.copytree(PKG / "csrc", self.pkg / "csrc")
        shutil.copy(PKG / "Makefile", self.pkg)
        shutil.copytree(ROOT / "include", tmp / "include")
        for header in ("torch/include/torch/csrc/autograd/python_variable.h", "python/Python.h"):
            (tmp / header).parent.mkdir(parents=True)
            (tmp / header).write_text("")
        out = 'while [ $# -gt 0 ]; do [ "$1" = -o ] && echo built > "$2"; shift; done\n'
        self.program("hipcc", out)
        self.program("cxx", f'echo "$@" >> {self.log}\n{out}')
        self.torch("1.0 abc")

    def program(self, name, text):
        p = self.tmp / name
        p.write_text("#!/bin/sh\n" + text)
        p.chmod(0o755)

    def torch(self, version):
        self.program("py", f"echo {self.tmp}/torch {self.tmp}/python {version} 0x1\n")

    def make(self, **change):
        args = {"HIPCC": self.tmp / "hipcc", "CXX": self.tmp / "cxx", "PYTHON": self.tmp / "py", **change}
        r = subprocess.run(["make", "-C", str(self.pkg), *(f"{k}={v}" for k, v in args.items())], capture_output=True, text=True, timeout=100)
        return r.returncode, r.stdout + r.stderr

    def builds(self):
        return self.log.read_text().splitlines() if self.log.exists() else []


@pytest.fixture
def tree(tmp_path):
    if shutil.which("make") is None:
        pytest.skip("make is not available")
    return Tree(tmp_path)


def test_the_extension_is_built_again_for_another_torch(tree):
    assert tree.make()[0] == 0 and len(tree.builds()) == 1
    assert '-DFDLLM_TORCH="1.0 abc"' in tree.builds()[0]
    assert tree.make()[0] == 0 and len(tree.builds()) == 1  # nothing has changed
    tree.torch("1.1 abd")
    assert tree.make()[0] == 0 and len(tree.builds()) == 2
    assert '-DFDLLM_TORCH="1.1 abd"' in tree.builds()[1]


def test_the_library_is_built_where_the_extension_cannot_be(tree):
    for missing in (dict(CXX=tree.tmp / "none"), dict(PYTHON=tree.tmp / "none"), "python/Python.h", "torch/include/torch/csrc/autograd/python_variable.h"):
        assert tree.make()[0] == 0 and (tree.pkg / "fdllm_calls.so").exists()
        (tree.pkg / "libfdllm.so").unlink()
        if isinstance(missing, dict):
            rc, text = tree.make(**missing)
        else:
            (tree.tmp / missing).rename(tree.tmp / "away")
            rc, text = tree.make()
            (tree.tmp / "away").rename(tree.tmp / missing)
        assert rc == 0 and "left out" in text, text
        assert (tree.pkg / "libfdllm.so").exists() and not (tree.pkg / "fdllm_calls.so").exists()  # (no older one either)


def test_an_error_in_compiling_the_extension_is_an_error(tree):
    tree.program("cxx", "exit 1\n")
    assert tree.make()[0] != 0


def test_build_takes_its_own_python(monkeypatch):
    import __graft_entry__ as entry

    seen = []
    monkeypatch.setattr(entry.subprocess, "run", lambda args, check: seen.append(args))
    entry.build()
    assert f"PYTHON={sys.executable}" in seen[0]
