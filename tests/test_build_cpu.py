"""The build script: what depends on what."""

import importlib.util
import stat
from pathlib import Path

import pytest

PKG_ROOT = Path(__file__).resolve().parents[1] / "breeze-tts-2_b200"


@pytest.fixture
def script(tmp_path):
    """build.py over a source tree of one small kernel."""
    spec = importlib.util.spec_from_file_location("breeze_b200_build_test", PKG_ROOT / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "one.cu").write_text('extern "C" int one() { return 1; }\n')
    mod.CSRC, mod.BUILD = tmp_path / "csrc", tmp_path / "_build"
    mod.OUT, mod.BIND_OUT = tmp_path / "lib.so", tmp_path / "bind.so"
    return mod


def _compiler(tmp_path, text):
    cxx = tmp_path / "cxx"
    cxx.write_text("#!/bin/sh\n" + text)
    cxx.chmod(cxx.stat().st_mode | stat.S_IXUSR)
    return str(cxx)


@pytest.mark.parametrize("cxx", ["echo no Python.h >&2; exit 1\n", None])
def test_the_library_does_not_need_the_bindings_headers(script, tmp_path, monkeypatch, cxx):
    monkeypatch.setenv("CXX", _compiler(tmp_path, cxx) if cxx else str(tmp_path / "nothing"))
    script.BIND_OUT.write_text("of an older build")
    with pytest.warns(UserWarning, match="no Python.h" if cxx else "nothing"):
        assert script.build(force=True) == script.OUT
    assert script.OUT.stat().st_size > 0 and not script.BIND_OUT.exists()
