"""build.py: the C library needs nothing but nvcc; the torch binding is built beside it where torch is there."""
import importlib.util
import os
import subprocess
import sys

import pytest

BUILD = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "vitni-tensor_b200", "build.py")


@pytest.fixture
def build(monkeypatch, tmp_path):
    """The module on files of its own: a library that is up to date and a binding that is not."""
    spec = importlib.util.spec_from_file_location("vtq_build", BUILD)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    lib, binding = tmp_path / "libvtq.so", tmp_path / "_serving.so"
    lib.write_text("built")
    binding.write_text("of an earlier build")
    os.utime(binding, (1, 1))
    monkeypatch.setattr(m, "OUT", str(lib))
    monkeypatch.setattr(m, "BINDING", str(binding))
    monkeypatch.setattr(m, "build", lambda **kw: str(lib))
    return m


def test_the_library_is_built_without_torch(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.main([]) == 0
    out = capsys.readouterr()
    assert build.OUT in out.out and "torch" in out.err
    assert not os.path.exists(build.BINDING)  # one of another build would not fit this library


def test_the_library_is_built_without_torchs_headers(build, monkeypatch, capsys):
    def fails(cmd, **kw):
        raise subprocess.CalledProcessError(1, cmd)

    monkeypatch.setattr(build.subprocess, "run", fails)
    assert build.main([]) == 0
    out = capsys.readouterr()
    assert build.OUT in out.out and "_serving.so" in out.err
    assert not os.path.exists(build.BINDING)


def test_both_where_both_can_be_built(build, monkeypatch, capsys):
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: open(build.BINDING, "w").write("new"))
    assert build.main([]) == 0
    assert capsys.readouterr().out.split("\n")[-3:-1] == [build.OUT, build.BINDING]
    assert open(build.BINDING).read() == "new"
