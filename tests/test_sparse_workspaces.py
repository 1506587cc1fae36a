"""A workspace sized for the largest call holds every smaller one (sizes alone: no
GPU): fewer tokens or positions may take another kernel, cut into more parts."""

import ctypes

import pytest

from molla_amd import _lib, gpu

TOKENS = [*range(1, 140), 200, 255, 256, 257, 300, 512, 1024, 2048]


def rises(sizes):
    most = 0
    for n in sizes:
        assert n >= most > -1 and n > 0
        most = n


def weight(kind, rows, cols):
    return _lib.MiWeight(1 << 20, kind, rows, cols, _lib.lib().mi_row_bytes(kind, cols))


@pytest.mark.parametrize("experts", [2, 8, 64, 128])
@pytest.mark.parametrize("width,hidden", [(256, 512), (256, 8192), (1024, 4096), (4096, 14336), (2048, 1024), (4096, 512)])
@pytest.mark.parametrize("kinds", [(12, 12), (12, 14), (14, 14), (8, 8)])
def test_experts(experts, width, hidden, kinds):
    L = _lib.lib()
    stack = experts * hidden
    d = _lib.MiExperts(experts, width, hidden, 0, weight(kinds[0], stack, width), weight(kinds[0], stack, width),
                       weight(kinds[1], experts * width, hidden))
    for used in (1, 2, 8):
        if used <= experts:
            rises(L.mi_experts_workspace(ctypes.byref(d), t, used) for t in TOKENS)
        rises(L.mi_experts_matmul_workspace(experts, width, used, t * used) for t in TOKENS)
    rises(L.mi_router_workspace(experts, t) for t in TOKENS)


@pytest.mark.parametrize("heads,kvh,d", [(32, 8, 128), (32, 4, 64), (8, 2, 96), (4, 2, 256), (8, 8, 64)])
@pytest.mark.parametrize("form", [gpu.CACHE_F16, gpu.CACHE_Q8])
@pytest.mark.parametrize("window,first", [(4096, 4), (1024, 64), (7, 0), (100000, 4)])
@pytest.mark.parametrize("one", [0, 1])
def test_window(heads, kvh, d, form, window, first, one):
    size = _lib.lib().mi_attend_window_workspace
    for count in (1, 100, 1000, 5000, 32768, 131072):
        rises(size(heads, kvh, d, form, window, first, count, t, one) for t in TOKENS)
    for t in (1, 2, 8, 9, 40, 256):
        rises(size(heads, kvh, d, form, window, first, count, t, one) for count in range(1, 140000, 397))


@pytest.mark.parametrize("experts,window,hidden", [(0, 512, 512), (0, 64, 512), (8, 0, 512), (8, 100, 4096),
                                                   (64, 0, 4096), (64, 512, 512)])
@pytest.mark.parametrize("form", [gpu.CACHE_F16, gpu.CACHE_Q8])
def test_layer_of_a_chunk(experts, window, hidden, form):
    """Above 8 tokens, as a prompt's chunks run on one workspace, the last one shorter."""
    d = _lib.MiLayerDesc()
    d.width, d.hidden, d.heads, d.kv_heads, d.head_dim, d.rope_dim = 1024, hidden, 8, 2, 128, 128
    d.eps, d.attn_scale, d.cache_form, d.window, d.first = 1e-5, 0.1, form, window, 4
    d.router = 1 << 20
    d.experts, d.experts_used, d.router_scale = experts, min(experts, 4), 1.0
    stack = max(experts, 1)
    d.gate = d.up = weight(12, stack * hidden, 1024)
    d.down = weight(12, stack * 1024, hidden)
    rises(_lib.lib().mi_layer_workspace(ctypes.byref(d), 8192, t) for t in TOKENS if t > 8)
