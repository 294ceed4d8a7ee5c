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
