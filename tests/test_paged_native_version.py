"""CPU: the native calls on a paged cache read tensors by the layouts of the torch they were built against, and call the library by its
signatures: with any others Python takes every call."""
import pytest
import torch

from pbs_attn_amd import _lib


def _loaded(monkeypatch):
    monkeypatch.setattr(_lib, "_paged_host", None)
    return _lib.paged_host()


def test_the_module_says_what_it_was_built_for(monkeypatch):
    host = _loaded(monkeypatch)
    assert host is not _lib._no_paged_host
    assert host.torch_version == str(torch.__version__) and host.abi_version == _lib.load().pbs_abi_version()


def test_another_torch(monkeypatch):
    monkeypatch.setattr(torch, "__version__", "2.9.1+rocm7.0")
    with pytest.warns(UserWarning, match="through Python.*2.9.1"):
        assert _loaded(monkeypatch) is _lib._no_paged_host


def test_another_library(monkeypatch):
    class Lib:
        def __getattr__(self, name):
            return getattr(lib, name)

        def pbs_abi_version(self):
            return lib.pbs_abi_version() + 1
    lib = _lib.load()
    monkeypatch.setattr(_lib, "_lib", Lib())
    with pytest.warns(UserWarning, match="through Python"):
        assert _loaded(monkeypatch) is _lib._no_paged_host
