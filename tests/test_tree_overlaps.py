"""The entry points of a step over drafted trees refuse outputs that lie among what
other blocks still read or write, before anything is queued (no GPU: every call here
returns from the checks of shim.cpp)."""

import ctypes

import pytest

from molla_amd import _lib
from tests.test_tree_refusals import ARG, FAKE, refused

F = 4  # bytes of a value


def qk(**change):
    """Three tokens of 8 over 2 heads of 64, q, k and v parts of a fused row of 768, its outputs apart."""
    q = FAKE
    d = dict(heads=8, kv_heads=2, head_dim=64, rope_dim=64, neox=1, tokens=3, eps=1e-5, q=q, k=q + 512 * F, v=q + 640 * F,
             q_stride=768, k_stride=768, v_stride=768, q_out=q + 4096 * F, q_out_stride=512, k_out=q + 8192 * F,
             k_out_stride=128, rope_steps=FAKE, pos=FAKE, k_cache=FAKE * 2, v_cache=FAKE * 3, cells=FAKE)
    return _lib.MiQk(**{**d, **change})


Q, K, V, QO, KO = FAKE, FAKE + 512 * F, FAKE + 640 * F, FAKE + 4096 * F, FAKE + 8192 * F


@pytest.mark.parametrize("change,text", [
    (dict(q_out=Q + 16), "q_out lies among the rows of q"),                             # shifted by a few values
    (dict(q_out=Q + 64 * F, q_out_stride=768), "q_out lies among the rows of q"),        # by a head, at the same stride
    (dict(q_out=Q - 511 * F, q_out_stride=768), "q_out lies among the rows of q"),
    (dict(q_out=Q + (2 * 768 + 511) * F), "q_out lies among the rows of q"),             # the last value
    (dict(q_out=Q - (2 * 512 + 511) * F), "q_out lies among the rows of q"),             # its own last value
    (dict(q_out=Q + 768 * F, q_out_stride=768), "q_out lies among the rows of q"),       # a row further
    (dict(q=QO + 9999 * F, q_out=K, q_out_stride=768), "q_out lies among the rows of k"),
    (dict(q=QO + 9999 * F, q_out=Q + 767 * F, q_out_stride=768), "q_out lies among the rows of v"),  # (v's last value)
    (dict(q=QO + 9999 * F, k=KO + 9999 * F, q_out=V, q_out_stride=768), "q_out lies among the rows of v"),
    (dict(k_out=Q + 256 * F, k_out_stride=768), "k_out lies among the rows of q"),
    (dict(k_out=K + 32 * F, k_out_stride=768), "k_out lies among the rows of k"),
    (dict(k_out=V, k_out_stride=768), "k_out lies among the rows of v"),
    (dict(k_out=V + 2 * 768 * F), "k_out lies among the rows of v"),
    (dict(k_out=QO + 512 * F), "k_out lies among the rows of q_out"),
    (dict(q_out=Q, q_out_stride=768, k_out=Q + 384 * F, k_out_stride=768), "k_out lies among the rows of q"),
    (dict(k=Q + 448 * F, q_out=Q, q_out_stride=768), "q_out lies among the rows of k"),  # in place over a shared part
    (dict(v_cache=FAKE * 2), "one cache")])
def test_qk_outputs_among_rows(change, text):
    refused(_lib.lib().mi_qk_norm_rope(None, ctypes.byref(qk(**change))), ARG, text)
