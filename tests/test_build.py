"""What the build makes where a host C++ compiler or Python's headers are missing, and for which Python. hipcc is a script here
that makes the file it is asked for."""
import os
import sys
import sysconfig

import pytest

from nunchi_amd import build as nb


@pytest.fixture
def places(tmp_path, monkeypatch):
    """Library and module in a folder of the test's own, one source, hipcc replaced."""
    fake = tmp_path / "hipcc"
    fake.write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\necho made > "$2"\n')
    fake.chmod(0o755)
    monkeypatch.setattr(nb, "HIPCC", str(fake))
    monkeypatch.setattr(nb, "SOURCES", nb.SOURCES[:1])
    monkeypatch.setattr(nb, "LIB", str(tmp_path / "libseoul_hip.so"))
    monkeypatch.setattr(nb, "MODULE", str(tmp_path / os.path.basename(nb.MODULE)))
    monkeypatch.delenv("CXX", raising=False)
    return tmp_path


def test_the_library_is_built_without_a_host_compiler(places, monkeypatch, capsys):
    monkeypatch.setenv("CXX", str(places / "no-such-compiler"))
    for name in ("_batch.so", os.path.basename(nb.MODULE)):    # what an earlier build left
        (places / name).write_text("old")
    assert nb.build() == nb.LIB and os.path.exists(nb.LIB)
    assert not [f for f in os.listdir(places) if f.startswith("_batch")], "an old module would be called with another library"
    assert "_batch" in capsys.readouterr().err


def test_the_library_is_built_without_pythons_headers(places, monkeypatch, capsys):
    monkeypatch.setattr(nb.sysconfig, "get_paths", lambda: {"include": str(places / "no-headers")})
    assert nb.build() == nb.LIB and os.path.exists(nb.LIB)
    assert "Python.h" in capsys.readouterr().err


def test_a_module_that_does_not_compile_is_an_error(places, monkeypatch):
    monkeypatch.setenv("CXX", "false")
    with pytest.raises(RuntimeError, match="_batch"):
        nb.build()


def test_the_module_is_this_pythons(places):
    """Its file name carries the interpreter's tag, so that another Python version does not load it."""
    nb.build()
    assert os.path.basename(nb.MODULE) == "_batch" + sysconfig.get_config_var("EXT_SUFFIX")
    assert os.path.exists(nb.MODULE)
    from nunchi_amd import _batch
    assert _batch.__file__.endswith(sysconfig.get_config_var("EXT_SUFFIX")) and sys.modules["nunchi_amd._batch"] is _batch
