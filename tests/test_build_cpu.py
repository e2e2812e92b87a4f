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


def test_the_bindings_follow_torch(script, tmp_path, monkeypatch):
    """Compiled again after torch was exchanged, and not before."""
    monkeypatch.setenv("CXX", _compiler(tmp_path, f'echo "$@" >> {tmp_path}/calls\ntouch {tmp_path}/bind.so\n'))
    calls = lambda: (tmp_path / "calls").read_text().splitlines()  # noqa: E731
    script.build()
    script.build()
    assert len(calls()) == 1 and f'BREEZE_TORCH_VERSION="{script.torch_version()}"' in calls()[0]
    monkeypatch.setattr(script, "torch_version", lambda: "99.0")
    script.build()
    script.build()
    assert len(calls()) == 2 and 'BREEZE_TORCH_VERSION="99.0"' in calls()[1]


def test_the_installed_torch_is_named_as_it_names_itself(script):
    import torch

    assert script.torch_version() == torch.__version__


@pytest.mark.parametrize("bind", [None, "other"])
def test_calls_without_fitting_bindings_go_through_python(bind, monkeypatch):
    import sys
    import types

    import breeze_b200
    import torch
    from breeze_b200.fused import paged

    made = None if bind is None else types.SimpleNamespace(torch_version="1.0", append=None, attention=None, bind=None)
    monkeypatch.setattr(paged, "_bound", None)
    monkeypatch.delattr(breeze_b200, "_paged_bind", raising=False)
    monkeypatch.setitem(sys.modules, "breeze_b200._paged_bind", made)
    row = torch.zeros(1, 64, dtype=torch.bfloat16)
    pages = torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.warns(RuntimeWarning, match="does not load"), pytest.raises(RuntimeError, match="CUDA tensors"):
        paged.paged_attention(row, pages, pages, one[None], one)
    with pytest.raises(RuntimeError, match="CUDA tensors"):  # said once
        paged.paged_attention(row, pages, pages, one[None], one)
