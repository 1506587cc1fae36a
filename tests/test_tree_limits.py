"""Sizes and values that the entry points of a step over drafted trees refuse at their
limits, before anything is queued (no GPU: every call here returns from the checks)."""

import ctypes

import pytest

from molla_amd import _lib
from tests.test_tree_refusals import ARG, ATTEND, FAKE, LAYER, TREE, layer_desc, refused


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_a_scale_that_is_not_finite(scale):
    tree = _lib.MiTree(**TREE, pos=FAKE, cells=FAKE)
    refused(_lib.lib().mi_attend_tree(*{**ATTEND, "scale": scale, "tree": ctypes.byref(tree)}.values()), ARG, "scale")
    desc = layer_desc(attn_scale=scale)
    refused(_lib.lib().mi_decoder_layer_tree(*{**LAYER, "desc": ctypes.byref(desc), "tree": ctypes.byref(tree)}.values()), ARG,
            "scale")
