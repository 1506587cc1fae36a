"""The header, the library and the bindings are of one version, and a library of another
is refused when it is loaded: a descriptor that grew would be read past its end."""

import ctypes
import os
import re

import pytest

from molla_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# sizes by version: one that changes here takes the next number
SIZES = {2: dict(MiWeight=32, MiLayerDesc=424, MiQk=184, MiTree=56, MiExperts=112)}


def text(*path):
    with open(os.path.join(ROOT, *path)) as f:
        return f.read()


def test_one_version():
    header = int(re.search(r"#define MI_VERSION (\d+)", text("include", "molla_mi.h")).group(1))
    mojo = int(re.search(r"comptime MI_VERSION = (\d+)", text("mojo", "molla_mi.mojo")).group(1))
    assert header == mojo == _lib.VERSION == _lib.lib().mi_version()


def test_structs_of_this_version():
    assert {n: ctypes.sizeof(getattr(_lib, n)) for n in SIZES[_lib.VERSION]} == SIZES[_lib.VERSION]


def test_another_version_is_refused(monkeypatch):
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "VERSION", _lib.VERSION - 1)
    with pytest.raises(RuntimeError, match="version"):
        _lib.lib()
    assert _lib._lib is None
