"""The decoder layer takes experts of every width that mi_experts takes: multiples of
64, of 256 where the down projection is of a K-quant (on the host: the call ends at its
workspace)."""

import ctypes

import pytest

from molla_amd import _lib
from tests.test_sparse_refusals import SHAPE, WORK, far, refused, weight


def layer(hidden, kinds, experts=4, **kw):
    d = _lib.MiLayerDesc()
    d.width, d.hidden, d.heads, d.kv_heads, d.head_dim, d.rope_dim = 256, hidden, 4, 2, 64, 64
    d.eps, d.attn_scale = 1e-5, 0.125
    d.attn_norm = d.ffn_norm = d.rope_steps = d.router = far(9)
    d.experts, d.experts_used, d.router_flags, d.router_scale = experts, 2, 2, 1.0
    n = experts or 1
    for name, (r, c, k) in dict(wq=(256, 256, 12), wk=(128, 256, 12), wv=(128, 256, 12), wo=(256, 256, 12),
                                gate=(n * hidden, 256, kinds[0]), up=(n * hidden, 256, kinds[0]),
                                down=(n * 256, hidden, kinds[1])).items():
        setattr(d, name, weight(r, c, kind=k) if hidden > 0 or name[0] == "w" else _lib.MiWeight())
    return _lib.lib().mi_decoder_layer(None, ctypes.byref(d), far(2), far(3), far(4), 0, far(5), 8, 1, far(6), 100)


@pytest.mark.parametrize("hidden,kinds", [(64, (12, 8)), (192, (8, 8)), (320, (12, 2)), (704, (14, 8)), (768, (12, 14)),
                                          (1408, (8, 6))])
def test_taken(hidden, kinds):
    refused(layer(hidden, kinds), WORK, "workspace")


@pytest.mark.parametrize("hidden,kinds,experts,words", [
    (96, (12, 8), 4, "hidden 96"), (0, (12, 8), 4, "hidden 0"), (-256, (12, 8), 4, "hidden -256"),
    (704, (12, 8), 0, "hidden 704"), (0, (12, 8), 0, "hidden 0")])
def test_refused(hidden, kinds, experts, words):
    refused(layer(hidden, kinds, experts), SHAPE, words)


def test_narrow_down_of_a_k_quant():
    d = _lib.MiExperts(4, 256, 704, 0, weight(2816, 256), weight(2816, 256, at=2), _lib.MiWeight(far(3), 12, 1024, 704, 396))
    rc = _lib.lib().mi_experts_mlp(None, ctypes.byref(d), far(4), 3, 2, far(5), far(6), far(7), 0, far(8), 1 << 30)
    refused(rc, SHAPE, "704 columns")
