"""Building the torch binding of the operators beside the library, with a stand-in for the compiler: no GPU, nothing of the package is touched."""
import os
import shutil
import stat
import subprocess
import warnings

import pytest

from omega_ai_b200 import native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_library_is_built_where_the_binding_cannot_be(monkeypatch):
    """A host that uses libomoe.so alone needs neither torch nor a C++ compiler."""
    native.build()
    for error in (ImportError("No module named 'torch'"), FileNotFoundError("g++"), subprocess.CalledProcessError(1, ["g++"])):
        def fails(force=False):
            raise error
        monkeypatch.setattr(native, "build_binding", fails)
        with pytest.warns(UserWarning, match="_torch_ops.so"):
            assert native.build() == os.path.join(ROOT, "omega_ai_b200", "libomoe.so")
    monkeypatch.undo()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        native.build()


@pytest.fixture
def package(tmp_path, monkeypatch):
    """A package folder of its own with a stand-in for the compiler: `write` is what it leaves at its -o, `status` its exit status."""
    pkg = tmp_path / "omega_ai_b200"
    pkg.mkdir()
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    monkeypatch.setattr(native, "_PKG", str(pkg))

    def compiler(write, status=0):
        cxx = tmp_path / "cxx"
        cxx.write_text('#!/bin/sh\nfor a in "$@"; do echo "$a" >> %s/args; done\nwhile [ "$1" != -o ]; do shift; done\nprintf %%s "%s" > "$2"\nexit %d\n'
                       % (tmp_path, write, status))
        cxx.chmod(cxx.stat().st_mode | stat.S_IXUSR)
        monkeypatch.setenv("CXX", str(cxx))

    return pkg, compiler


def later(path):
    """Newer than any source."""
    at = max(os.path.getmtime(os.path.join(native.CSRC, "bind", "torch_ops.cpp")), path.stat().st_mtime) + 100
    os.utime(path, (at, at))


def test_a_binding_for_another_torch_is_built_again(package):
    import torch

    pkg, compiler = package
    so = pkg / "_torch_ops.so"
    so.write_text("built for another torch")
    later(so)
    compiler("new")
    assert native.build_binding() == str(so)
    assert so.read_text() == "new"
    # one for the installed torch and Python stays: the compiler is given the mark that it has to carry
    given = [a for a in (pkg.parent / "args").read_text().splitlines() if torch.__version__ in a]
    assert len(given) == 1
    so.write_text("code " + given[0].split("=", 1)[1].strip('"') + " code")
    later(so)
    compiler("newer")
    native.build_binding()
    assert so.read_text() != "newer"


def test_the_built_binding_carries_its_mark():
    native.build()
    path = native.build_binding()
    before = os.stat(path).st_mtime_ns
    assert native.build_binding() == path and os.stat(path).st_mtime_ns == before
    assert native.binding_mark().encode() in open(path, "rb").read()


def test_a_build_that_fails_leaves_the_binding_alone(package):
    """The file appears whole or not at all: a process that loads it meanwhile, or after a failed build, does not find half of one."""
    pkg, compiler = package
    so = pkg / "_torch_ops.so"
    so.write_text("whole")
    compiler("half", status=1)
    with pytest.raises(subprocess.CalledProcessError):
        native.build_binding(force=True)
    assert so.read_text() == "whole" and [p.name for p in pkg.iterdir()] == ["_torch_ops.so"]
    compiler("next")
    with open(so) as held:  # as a process that has it loaded
        native.build_binding(force=True)
        assert held.read() == "whole" and so.read_text() == "next"
    assert [p.name for p in pkg.iterdir()] == ["_torch_ops.so"]
