"""Workspace sizes of windowed attention and of layers with a window, at shapes and
counts that no call can have: asked for on the host, none of them ends the process."""

import ctypes
import subprocess
import sys

import pytest

from molla_amd import _lib

ASK = """
import ctypes
from molla_amd import _lib
d = _lib.MiLayerDesc()
d.width, d.hidden, d.heads, d.kv_heads, d.head_dim, d.rope_dim = 256, 512, 4, 2, 64, 64
d.window, d.first = 5, 1
d.{field} = {value}
print([_lib.lib().mi_layer_workspace(ctypes.byref(d), 100, t) for t in (1, 8, 9, 300)])
"""


@pytest.mark.parametrize("field,value", [("kv_heads", 0), ("kv_heads", -2), ("heads", 0), ("heads", 3), ("head_dim", 0),
                                         ("head_dim", 20), ("kv_heads", 3)])
def test_a_layer_that_cannot_be(field, value):
    r = subprocess.run([sys.executable, "-c", ASK.format(field=field, value=value)], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr)
    assert r.stdout.strip() == "[0, 0, 0, 0]"


def test_a_layer_that_can():
    d = _lib.MiLayerDesc()
    d.width, d.hidden, d.heads, d.kv_heads, d.head_dim, d.rope_dim, d.window = 256, 512, 4, 2, 64, 64, 5
    assert all(_lib.lib().mi_layer_workspace(ctypes.byref(d), 100, t) > 0 for t in (1, 8, 9, 300))
