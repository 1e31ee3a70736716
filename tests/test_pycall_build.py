"""The extension module of the chunk operators' Python calls is used by the
Python and the torch it was built with, and by no other: it reads tensors by
their layout in memory."""
import os

import pytest
import torch


@pytest.fixture(scope="module", autouse=True)
def built():
    from kyro_b200 import build
    build.build()


def _loaded(monkeypatch):
    """What a fresh process would load."""
    from kyro_b200 import _lib
    monkeypatch.setattr(_lib, "_calls", None)
    try:
        return _lib.calls()
    except ImportError:
        return None


def test_the_module_is_the_one_of_this_torch(monkeypatch):
    from kyro_b200 import build
    m = _loaded(monkeypatch)
    assert os.path.samefile(m.__file__, build.pycall_path(torch.__version__))
    assert m.chunk_attention


def test_a_module_of_another_torch_is_not_loaded(monkeypatch):
    monkeypatch.setattr(torch, "__version__", "2.12.1+cu999")
    assert _loaded(monkeypatch) is None


def test_a_module_of_another_python_is_not_loaded(monkeypatch):
    import sysconfig
    monkeypatch.setitem(sysconfig.get_config_vars(), "EXT_SUFFIX",
                        ".cpython-399-x86_64-linux-gnu.so")
    assert _loaded(monkeypatch) is None


def test_a_change_of_torch_builds_the_module_anew(monkeypatch, tmp_path):
    """(the compiler's stand-in writes the file it is asked for)"""
    from kyro_b200 import build
    fake = tmp_path / "cxx"
    fake.write_text("#!/bin/sh\nwhile [ \"$1\" != -o ]; do shift; done\necho built > \"$2\"\n")
    fake.chmod(0o755)
    monkeypatch.setenv("CXX", str(fake))
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    there = build.pycall_path(torch.__version__)
    build._build_pycall(False, False)
    assert set(os.listdir(tmp_path)) == {"cxx", os.path.basename(there)}
    stamp = os.stat(there).st_mtime_ns
    build._build_pycall(False, False)
    assert os.stat(there).st_mtime_ns == stamp  # up to date
    monkeypatch.setattr(build.runpy, "run_path", lambda path: {"__version__": "9.9"})
    build._build_pycall(False, False)
    assert os.path.exists(build.pycall_path("9.9"))
