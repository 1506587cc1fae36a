"""What the router, the experts' products and MLP, windowed attention and the layer
with them refuse, before anything is queued (no GPU: every call returns from the
checks)."""

import ctypes

import pytest

from molla_amd import _lib

FAKE = 0x100000  # never dereferenced
BIG = 1 << 40
ARG, KIND, SHAPE, WORK, ALIGN = -1, -2, -3, -4, -6


def far(i):
    return FAKE + i * BIG


def refused(rc, code, words):
    msg = _lib.lib().mi_last_error().decode()
    assert rc == code, (rc, msg)
    assert words in msg, msg


def router(**kw):
    a = dict(x=far(1), router=far(2), bias=None, width=256, experts=8, used=2, tokens=4, flags=0, scale=1.0, ids=far(3),
             weights=far(4), work=far(5), bytes=1 << 20)
    a.update(kw)
    return _lib.lib().mi_router(None, *a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(x=None), ARG, "null"), (dict(router=None), ARG, "null"), (dict(ids=None), ARG, "null"),
    (dict(weights=None), ARG, "null"), (dict(width=254), SHAPE, "254"), (dict(width=0), SHAPE, "0 values"),
    (dict(experts=0), SHAPE, "0 experts"), (dict(experts=513), SHAPE, "513"), (dict(used=0), SHAPE, "0 of 8"),
    (dict(used=9), SHAPE, "9 of 8"), (dict(experts=100, used=65), SHAPE, "65"), (dict(tokens=0), ARG, "tokens 0"),
    (dict(tokens=65537), ARG, "65537"), (dict(flags=4), ARG, "0x4"), (dict(scale=float("nan")), ARG, "scale"),
    (dict(scale=float("inf")), ARG, "scale"), (dict(x=far(1) + 4), ALIGN, "input"), (dict(router=far(2) + 8), ALIGN, "router"),
    (dict(weights=far(3) + 16), ARG, "lies in"), (dict(bias=far(3)), ARG, "lies in"), (dict(work=None), WORK, "workspace"),
    (dict(work=far(5) + 16), WORK, "workspace"), (dict(bytes=255), WORK, "255"), (dict(work=far(1)), ARG, "lies in"),
    (dict(work=far(3)), ARG, "lies in"), (dict(bias=far(5)), ARG, "lies in")])
def test_router(kw, code, words):
    refused(router(**kw), code, words)


def matmul(**kw):
    a = dict(kind=12, w=far(1), row_bytes=144, experts=4, rows=64, cols=256, x=far(2), share=2, ids=far(3), pairs=8,
             y=far(4), work=far(5), bytes=1 << 30)
    a.update(kw)
    return _lib.lib().mi_experts_matmul(None, *a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(kind=1), KIND, "type 1"), (dict(w=None), ARG, "null"), (dict(x=None), ARG, "null"), (dict(ids=None), ARG, "null"),
    (dict(y=None), ARG, "null"), (dict(row_bytes=288), SHAPE, "row_bytes"), (dict(cols=128), SHAPE, "128 columns"),
    (dict(rows=0), SHAPE, "0 rows"), (dict(rows=-4), SHAPE, "-4 rows"), (dict(experts=0), SHAPE, "0 experts"),
    (dict(experts=513), SHAPE, "513"), (dict(experts=512, rows=1 << 23), SHAPE, "too many"), (dict(pairs=0), SHAPE, "0 rows"),
    (dict(pairs=(1 << 20) + 2), SHAPE, "1048578"), (dict(share=3), SHAPE, "3 for each"), (dict(share=0), SHAPE, "0 for each"),
    (dict(w=far(1) + 4), ALIGN, "aligned"), (dict(kind=8, cols=64, row_bytes=68, w=far(1) + 4), ALIGN, "16-byte"),
    (dict(x=far(2) + 4), ALIGN, "input"), (dict(y=far(4) + 4), ALIGN, "output"), (dict(y=far(2)), ARG, "lies in"),
    (dict(y=far(3) - 16), ARG, "lies in"), (dict(y=far(1) + 64), ARG, "lies in"), (dict(work=None), WORK, "workspace"),
    (dict(work=far(5) + 8), WORK, "workspace"), (dict(bytes=4095), WORK, "4096 needed"), (dict(work=far(2)), ARG, "workspace lies"),
    (dict(work=far(4)), ARG, "workspace lies"), (dict(work=far(3)), ARG, "workspace lies")])
def test_matmul(kw, code, words):
    refused(matmul(**kw), code, words)


def weight(rows, cols, kind=12, at=1, **kw):
    w = _lib.MiWeight(far(at), kind, rows, cols, _lib.lib().mi_row_bytes(kind, cols))
    for k, v in kw.items():
        setattr(w, k, v)
    return w


def experts(**kw):
    d = _lib.MiExperts(4, 256, 512, 0, weight(2048, 256), weight(2048, 256, at=2), weight(1024, 512, at=3))
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def mlp(desc=None, **kw):
    a = dict(d=ctypes.byref(desc or experts()), x=far(4), tokens=3, used=2, ids=far(5), weights=far(6), out=far(7), epi=0,
             work=far(8), bytes=1 << 30)
    a.update(kw)
    return _lib.lib().mi_experts_mlp(None, *a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(d=None), ARG, "null"), (dict(x=None), ARG, "null"), (dict(ids=None), ARG, "null"), (dict(weights=None), ARG, "null"),
    (dict(out=None), ARG, "null"), (dict(tokens=0), ARG, "tokens 0"), (dict(tokens=65537), ARG, "65537"),
    (dict(used=0), SHAPE, "0 experts a token"), (dict(used=65), SHAPE, "65"), (dict(tokens=65536, used=17), SHAPE, "rows"),
    (dict(epi=1), ARG, "epilogue"), (dict(epi=4), ARG, "epilogue"), (dict(x=far(4) + 4), ALIGN, "input"),
    (dict(out=far(7) + 8), ALIGN, "output"), (dict(out=far(5)), ARG, "lies in"), (dict(out=far(6) - 16), ARG, "lies in"),
    (dict(work=None), WORK, "workspace"), (dict(work=far(8) + 4), WORK, "workspace"), (dict(bytes=1000), WORK, "1000"),
    (dict(work=far(4)), ARG, "workspace lies"), (dict(work=far(7)), ARG, "workspace lies")])
def test_mlp(kw, code, words):
    refused(mlp(**kw), code, words)


@pytest.mark.parametrize("kw,code,words", [
    (dict(experts=0), SHAPE, "0 experts"), (dict(width=0), SHAPE, "width 0"), (dict(hidden=100), SHAPE, "hidden 100"),
    (dict(act=3), ARG, "act 3"), (dict(hidden=256), SHAPE, "gate"), (dict(up=weight(1024, 256)), SHAPE, "up"),
    (dict(down=weight(512, 512)), SHAPE, "down"), (dict(up=weight(2048, 256, kind=14)), KIND, "type 12"),
    (dict(gate=weight(2048, 256, data=None)), ARG, "null"), (dict(gate=weight(2048, 256, kind=99)), KIND, "99"),
    (dict(down=weight(1024, 512, kind=8, data=far(3) + 4)), ALIGN, "16-byte")])
def test_mlp_descriptor(kw, code, words):
    refused(mlp(experts(**kw)), code, words)


def window(**kw):
    a = dict(form=0, q=far(1), q_stride=1024, k=far(2), v=far(3), cache_stride=1 << 20, index=None, index_stride=0, heads=8,
             kv_heads=2, head_dim=128, scale=0.1, window=100, first=4, pos=far(4), max_count=500, tokens=3, out=far(5),
             work=far(6), bytes=1 << 30)
    a.update(kw)
    return _lib.lib().mi_attend_window(None, *a.values())


@pytest.mark.parametrize("kw,code,words", [
    (dict(q=None), ARG, "null"), (dict(k=None), ARG, "null"), (dict(v=None), ARG, "null"), (dict(pos=None), ARG, "null"),
    (dict(out=None), ARG, "null"), (dict(heads=6), SHAPE, "3 query heads"), (dict(heads=9), SHAPE, "9 query heads"),
    (dict(kv_heads=0), SHAPE, "0 key heads"), (dict(head_dim=100), SHAPE, "100"), (dict(head_dim=544), SHAPE, "544"),
    (dict(heads=1 << 15, kv_heads=1 << 14, q_stride=1 << 24), SHAPE, "rows of"), (dict(form=2), SHAPE, "form 2"),
    (dict(window=0), ARG, "window of 0"), (dict(window=-1), ARG, "window of -1"), (dict(first=-1), ARG, "first -1"),
    (dict(max_count=0), SHAPE, "max_count"), (dict(tokens=0), ARG, "tokens 0"), (dict(tokens=65537), ARG, "65537"),
    (dict(scale=float("inf")), ARG, "scale"), (dict(scale=float("nan")), ARG, "scale"), (dict(q_stride=1020), SHAPE, "stride"),
    (dict(q_stride=1026), ALIGN, "16-byte"), (dict(q=far(1) + 4), ALIGN, "queries"), (dict(out=far(5) + 4), ALIGN, "output"),
    (dict(cache_stride=500 * 256 - 8), SHAPE, "fewer than 500"), (dict(cache_stride=-8), SHAPE, "negative"),
    (dict(cache_stride=(1 << 20) + 4), ALIGN, "multiple of 8"), (dict(k=far(2) + 8), ALIGN, "caches"),
    (dict(v=far(3) + 2), ALIGN, "caches"), (dict(index=far(7), index_stride=499), SHAPE, "fewer than 500"),
    (dict(index=far(7), index_stride=-1), SHAPE, "negative"), (dict(out=far(1)), ARG, "among the queries"),
    (dict(out=far(1) + 4096 * 2), ARG, "among the queries"), (dict(work=None), WORK, "workspace"),
    (dict(work=far(6) + 4), WORK, "workspace"), (dict(bytes=1000), WORK, "1000")])
def test_window(kw, code, words):
    refused(window(**kw), code, words)


def layer(**kw):
    d = _lib.MiLayerDesc()
    d.width, d.hidden, d.heads, d.kv_heads, d.head_dim, d.rope_dim = 256, 512, 4, 2, 64, 64
    d.eps, d.attn_scale = 1e-5, 0.125
    d.attn_norm = d.ffn_norm = d.rope_steps = d.router = far(9)
    d.experts, d.experts_used, d.router_flags, d.router_scale = 4, 2, 2, 1.0
    for n, (r, c) in dict(wq=(256, 256), wk=(128, 256), wv=(128, 256), wo=(256, 256), gate=(2048, 256), up=(2048, 256),
                          down=(1024, 512)).items():
        setattr(d, n, weight(r, c))
    resid, tokens = kw.pop("resid", far(2)), kw.pop("tokens", 1)
    for k, v in kw.items():
        setattr(d, k, v)
    return _lib.lib().mi_decoder_layer(None, ctypes.byref(d), resid, far(3), far(4), 0, far(5), 8, tokens, far(6), 100)


@pytest.mark.parametrize("kw,code,words", [
    (dict(), WORK, "workspace"),  # (all but the workspace is in order)
    (dict(experts=0, gate=weight(512, 256), up=weight(512, 256), down=weight(256, 512), router=None), WORK, "workspace"),
    (dict(experts=-1), SHAPE, "-1 experts"), (dict(experts=600), SHAPE, "600"), (dict(experts=5), SHAPE, "gate"),
    (dict(experts_used=0), SHAPE, "0 of 4"), (dict(experts_used=5), SHAPE, "5 of 4"), (dict(router=None), ARG, "router"),
    (dict(router=far(9) + 4), ALIGN, "router"), (dict(router_flags=8), ARG, "0x8"), (dict(router_scale=float("nan")), ARG, "scale"),
    (dict(ungated=1), ARG, "without a gate"), (dict(window=-1), ARG, "window of -1"), (dict(first=-2), ARG, "first -2"),
    (dict(up=weight(2048, 256, kind=13)), KIND, "type 13"), (dict(resid=far(2) + 4), ALIGN, "residual")])
def test_layer(kw, code, words):
    refused(layer(**kw), code, words)


def test_workspaces_of_what_is_refused_are_none():
    L = _lib.lib()
    assert L.mi_router_workspace(0, 1) == 0 and L.mi_router_workspace(8, 65537) == 0 and L.mi_router_workspace(8, 3) == 256
    assert L.mi_experts_matmul_workspace(4, 250, 1, 4) == 0 and L.mi_experts_matmul_workspace(4, 256, 3, 4) == 0
    assert L.mi_experts_workspace(None, 1, 1) == 0 and L.mi_experts_workspace(ctypes.byref(experts()), 65536, 64) == 0
    assert L.mi_attend_window_workspace(8, 2, 128, 0, 0, 0, 100, 1, 0) == 0
    d = _lib.MiLayerDesc()
    d.experts = 3
    assert L.mi_layer_workspace(ctypes.byref(d), 8, 1) == 0


def test_workspaces_hold_the_largest_calls():
    """Sizes of calls at the limits count past 32 bits."""
    L = _lib.lib()
    d = _lib.MiExperts(512, 4096, 14336, 0)
    pairs = 65536 * 16
    assert L.mi_experts_workspace(ctypes.byref(d), 65536, 16) > pairs * 14336 * 8
    assert L.mi_experts_matmul_workspace(512, 16384, 1, 1 << 20) > (1 << 20) * 16384 * 4
    assert L.mi_attend_window_workspace(32, 8, 128, 0, 4096, 4, 1 << 20, 65536, 0) >= 65536 * 32 * 128 * 4
