"""Building and loading the host module: a module of other sources is never loaded, and the CUDA library
does not wait for torch's headers."""

from __future__ import annotations

import shutil

import pytest

from lnet_b200 import _native
from lnet_b200 import build as _build


@pytest.fixture
def copy_of_the_module(tmp_path, monkeypatch):
    """The built module and what it was built from, at another place."""
    _native.native()
    lib = tmp_path / "_lib"
    lib.mkdir()
    for p in _build.LIB_DIR.glob("_torch_ops*"):
        shutil.copy(p, lib / p.name)
    source = tmp_path / "torch_ops.cpp"
    shutil.copy(_build.TORCH_OPS_SOURCE, source)
    monkeypatch.setattr(_build, "LIB_DIR", lib)
    monkeypatch.setattr(_build, "TORCH_OPS", lib / _build.TORCH_OPS.name)
    monkeypatch.setattr(_build, "TORCH_OPS_SOURCE", source)
    return source


def test_the_same_sources_are_not_stale_whatever_their_times(copy_of_the_module):
    assert not _build.torch_ops_stale()
    copy_of_the_module.touch()  # copied or checked out later: the same text
    assert not _build.torch_ops_stale()


def test_other_sources_and_another_torch_are_stale(copy_of_the_module, monkeypatch):
    import torch

    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "0.0.1")
        assert _build.torch_ops_stale()
    with open(copy_of_the_module, "a") as f:
        f.write("// changed\n")
    assert _build.torch_ops_stale()


def test_a_stale_module_that_cannot_be_rebuilt_is_an_error(copy_of_the_module, monkeypatch):
    with open(copy_of_the_module, "a") as f:
        f.write("#error\n")
    monkeypatch.setattr(_native, "_module", None)
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
        _native.native()


def test_the_cuda_library_is_built_without_torch_headers(monkeypatch, tmp_path):
    def no_headers(*_):
        raise RuntimeError("no torch headers")

    monkeypatch.setattr(_build, "build_torch_ops", no_headers)
    monkeypatch.setattr(_build, "LIB", tmp_path / "lib.so")
    monkeypatch.setattr(_build, "LIB_DIR", tmp_path)
    monkeypatch.setattr(_build, "ROOT", tmp_path)
    source = tmp_path / "empty.cu"
    source.write_text("extern \"C\" int lnet_empty() { return 0; }\n")
    monkeypatch.setattr(_build, "_sources", lambda: [source])
    with pytest.raises(RuntimeError, match="no torch headers"):
        _build.build()
    assert (tmp_path / "lib.so").exists()
