"""The CPython module of the list operators (csrc/gs_host.cpp) and the library that it calls belong to one header."""
import sys
import types

import pytest

import taichi_3d_gaussian_splatting_amd as package
from taichi_3d_gaussian_splatting_amd import _lib


def test_the_built_module_was_compiled_from_this_header():
    assert _lib.host().ABI_VERSION == _lib.ABI_VERSION


@pytest.mark.parametrize("version", [None, _lib.ABI_VERSION - 1, _lib.ABI_VERSION + 1])
def test_a_module_of_another_header_is_refused_before_it_is_bound(monkeypatch, version):
    """An older build would hand its arguments to other places of the library's functions."""
    bound = []
    other = types.ModuleType("_gs_host")
    other.bind = lambda *addresses: bound.append(addresses)
    if version is not None:
        other.ABI_VERSION = version
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setitem(sys.modules, package.__name__ + "._gs_host", other)
    monkeypatch.setattr(package, "_gs_host", other, raising=False)
    with pytest.raises(RuntimeError, match="_gs_host.*ABI"):
        _lib.host()
    assert not bound and _lib._host is None
