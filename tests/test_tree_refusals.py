"""The entry points of a step over drafted trees refuse bad arguments before
anything is queued (every call here returns from the checks of shim.cpp; no
GPU), and their structs lie in the Mojo binding as in C."""

import ctypes
import os
import re

import pytest

from molla_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x100000  # never dereferenced: every call below is refused first
ARG, SHAPE, WORKSPACE, ALIGN = -1, -3, -4, -6


def refused(rc, code, text):
    assert rc == code and text in _lib.lib().mi_last_error().decode(), (rc, _lib.lib().mi_last_error())


PAGE = dict(stream=None, batch=4, page=16, lengths=FAKE, news=FAKE, table=FAKE, table_stride=8, free_pages=FAKE,
            free_size=10, free_count=FAKE, free_left=FAKE + 64, kv_index=FAKE, index_stride=128, max_tokens=16,
            starts=FAKE, seq=None, pos=None, cells=FAKE)


@pytest.mark.parametrize("change,code,text", [
    (dict(lengths=None), ARG, "null"), (dict(news=None), ARG, "null"), (dict(table=None), ARG, "null"),
    (dict(free_count=None), ARG, "null"), (dict(free_left=None), ARG, "null"), (dict(starts=None), ARG, "null"),
    (dict(cells=None), ARG, "null"), (dict(batch=0), SHAPE, "batch"), (dict(batch=4097), SHAPE, "batch"),
    (dict(page=0), SHAPE, "pages"), (dict(table_stride=0), SHAPE, "pages"), (dict(free_size=-1), ARG, "free list"),
    (dict(free_pages=None), ARG, "free list"), (dict(free_left=FAKE), ARG, "free_left"),
    (dict(free_left=FAKE - 4), ARG, "free_left"), (dict(index_stride=0), SHAPE, "stride"),
    (dict(max_tokens=0), SHAPE, "max_tokens"), (dict(max_tokens=(1 << 30) + 1), SHAPE, "max_tokens")])
def test_page_plan_refusals(change, code, text):
    refused(_lib.lib().mi_page_plan(*{**PAGE, **change}.values()), code, text)


TREE_PLAN = dict(stream=None, batch=2, starts=FAKE, lengths=FAKE, parents=FAKE, max_nodes=8, tokens=16, pos=FAKE, mask=FAKE)


@pytest.mark.parametrize("change,code,text", [
    (dict(starts=None), ARG, "null"), (dict(lengths=None), ARG, "null"), (dict(parents=None), ARG, "null"),
    (dict(mask=None), ARG, "null"), (dict(batch=0), SHAPE, "batch"), (dict(max_nodes=0), SHAPE, "nodes"),
    (dict(max_nodes=257), SHAPE, "nodes"), (dict(tokens=0), SHAPE, "rows")])
def test_tree_plan_refusals(change, code, text):
    refused(_lib.lib().mi_tree_plan(*{**TREE_PLAN, **change}.values()), code, text)


def test_tree_words():
    words = _lib.lib().mi_tree_words
    assert [words(n) for n in (0, 1, 32, 33, 256, 257)] == [-1, 1, 1, 2, 8, -1]


QK = dict(heads=8, kv_heads=2, head_dim=64, rope_dim=64, neox=1, cache_form=0, tokens=3, eps=1e-5, q=FAKE, k=FAKE, v=FAKE,
          q_stride=768, k_stride=768, v_stride=768, q_out=FAKE + 64, q_out_stride=512, rope_steps=FAKE, pos=FAKE,
          k_cache=FAKE, v_cache=FAKE, cells=FAKE)


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), ARG, "null"), (dict(k=None), ARG, "null"), (dict(q_out=None), ARG, "null"),
    (dict(rope_steps=None), ARG, "null"), (dict(pos=None), ARG, "null"), (dict(v=None), ARG, "together"),
    (dict(cells=None), ARG, "together"), (dict(k_cache=None), ARG, "together"), (dict(q_norm=FAKE), ARG, "norms"),
    (dict(q_norm=FAKE, k_norm=FAKE, eps=0.0), ARG, "epsilon"),
    (dict(q_norm=FAKE, k_norm=FAKE, eps=float("nan")), ARG, "epsilon"), (dict(neox=2), ARG, "neox"),
    (dict(heads=6, kv_heads=2), SHAPE, "1, 2, 4 or 8"), (dict(head_dim=48), SHAPE, "multiple of 32"),
    (dict(head_dim=544), SHAPE, "512"), (dict(rope_dim=0), SHAPE, "rotary"), (dict(rope_dim=63), SHAPE, "rotary"),
    (dict(rope_dim=66), SHAPE, "rotary"), (dict(tokens=0), SHAPE, "tokens"), (dict(q_stride=511), SHAPE, "stride"),
    (dict(q_out_stride=511), SHAPE, "stride"), (dict(k_stride=127), SHAPE, "stride"), (dict(v_stride=127), SHAPE, "stride"),
    (dict(k_out=FAKE + 64, k_out_stride=127), SHAPE, "stride"), (dict(q_out=FAKE), SHAPE, "in place"),
    (dict(k_out=FAKE, k_out_stride=128), SHAPE, "in place"), (dict(cache_form=2), SHAPE, "form"),
    (dict(k_cache=FAKE + 8), ALIGN, "16-byte"), (dict(v_cache=FAKE + 2), ALIGN, "16-byte")])
def test_qk_refusals(change, code, text):
    d = _lib.MiQk(**{**QK, **change})
    refused(_lib.lib().mi_qk_norm_rope(None, ctypes.byref(d)), code, text)


def test_qk_refuses_no_descriptor():
    refused(_lib.lib().mi_qk_norm_rope(None, None), ARG, "null")


TREE = dict(batch=3, tokens=24, max_nodes=8, max_count=100, starts=FAKE, lengths=FAKE, mask=FAKE)
ATTEND = dict(stream=None, form=0, q=FAKE, q_stride=512, k_cache=FAKE, v_cache=FAKE, cache_stride=12800, kv_index=None,
              index_stride=0, heads=8, kv_heads=2, head_dim=64, scale=0.125, tree=None, out=FAKE + 24 * 2048, work=FAKE,
              work_bytes=1 << 30)


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), ARG, "null"), (dict(k_cache=None), ARG, "null"), (dict(v_cache=None), ARG, "null"),
    (dict(out=None), ARG, "null"), (dict(heads=12, kv_heads=4), SHAPE, "1, 2, 4 or 8"),
    (dict(head_dim=40), SHAPE, "multiple of 32"), (dict(form=2), SHAPE, "form"), (dict(q_stride=511), SHAPE, "stride"),
    (dict(cache_stride=12799), SHAPE, "fewer"), (dict(kv_index=FAKE, index_stride=99), SHAPE, "fewer"),
    (dict(q=FAKE + 4), ALIGN, "16-byte"), (dict(q_stride=514), ALIGN, "16-byte"), (dict(cache_stride=12804), ALIGN, "16-byte"),
    (dict(out=FAKE + 8), ALIGN, "16-byte"), (dict(work=None), WORKSPACE, "workspace"),
    (dict(out=FAKE), ARG, "among"), (dict(out=FAKE + 24 * 2048 - 16), ARG, "among"), (dict(out=FAKE - 24 * 2048 + 16), ARG, "among"),
    (dict(work=FAKE + 16), WORKSPACE, "workspace"), (dict(work_bytes=64), WORKSPACE, "needed"),
    (dict(tree=dict(starts=None)), ARG, "trees"), (dict(tree=dict(lengths=None)), ARG, "trees"),
    (dict(tree=dict(mask=None)), ARG, "trees"), (dict(tree=dict(batch=0)), SHAPE, "sequences"),
    (dict(tree=dict(tokens=0)), SHAPE, "sequences"), (dict(tree=dict(max_nodes=0)), SHAPE, "nodes"),
    (dict(tree=dict(max_nodes=257)), SHAPE, "nodes"), (dict(tree=dict(max_count=0)), SHAPE, "max_count")])
def test_attend_refusals(change, code, text):
    tree = _lib.MiTree(**{**TREE, **(change.get("tree") or {})})
    args = {**ATTEND, **change, "tree": ctypes.byref(tree)}
    refused(_lib.lib().mi_attend_tree(*args.values()), code, text)


@pytest.mark.parametrize("tree", [dict(batch=1, max_nodes=256, max_count=2 ** 31 - 1), dict(batch=40000, max_nodes=256, max_count=2 ** 20),
                                  dict(batch=10 ** 6, max_nodes=256, max_count=1)])
def test_attend_refuses_more_work_than_32_bits_count(tree):
    tree = _lib.MiTree(**{**TREE, **tree})
    args = {**ATTEND, "heads": 64, "kv_heads": 64, "q_stride": 4096, "kv_index": FAKE, "index_stride": 2 ** 31, "out": FAKE << 8,
            "work_bytes": 1 << 50, "tree": ctypes.byref(tree)}
    refused(_lib.lib().mi_attend_tree(*args.values()), SHAPE, "too much work")


def test_layer_refuses_it_before_its_first_launch():
    tree = _lib.MiTree(**{**TREE, "batch": 200000, "max_nodes": 256, "max_count": 2 ** 20, "pos": FAKE, "cells": FAKE})
    args = {**LAYER, "kv_index": FAKE, "index_stride": 2 ** 20, "work_bytes": 1 << 50, "desc": ctypes.byref(layer_desc()),
            "tree": ctypes.byref(tree)}
    refused(_lib.lib().mi_decoder_layer_tree(*args.values()), SHAPE, "too much work")


def test_attend_refuses_no_trees():
    refused(_lib.lib().mi_attend_tree(*ATTEND.values()), ARG, "trees")


def layer_desc(**change):
    d = _lib.MiLayerDesc(width=512, hidden=1024, heads=8, kv_heads=2, head_dim=64, rope_dim=64, eps=1e-5, attn_scale=0.125,
                         attn_norm=FAKE, ffn_norm=FAKE, rope_steps=FAKE)
    for name, rows, cols in (("wq", 512, 512), ("wk", 128, 512), ("wv", 128, 512), ("wo", 512, 512), ("gate", 1024, 512),
                             ("up", 1024, 512), ("down", 512, 1024)):
        setattr(d, name, _lib.MiWeight(FAKE, 12, rows, cols, cols // 256 * 144))
    for name, value in change.items():
        setattr(d, name, value)
    return d


LAYER = dict(stream=None, desc=None, resid=FAKE, k_cache=FAKE, v_cache=FAKE, cache_stride=12800, kv_index=None,
             index_stride=0, tree=None, work=FAKE, work_bytes=1 << 30)


@pytest.mark.parametrize("change,code,text", [
    (dict(resid=None), ARG, "null"), (dict(k_cache=None), ARG, "null"), (dict(v_cache=None), ARG, "null"),
    (dict(desc=dict(heads=12)), SHAPE, "1, 2, 4 or 8"), (dict(desc=dict(cache_form=3)), SHAPE, "form"),
    (dict(desc=dict(q_norm=FAKE)), ARG, "together"), (dict(cache_stride=12799), SHAPE, "fewer"),
    (dict(kv_index=FAKE, index_stride=99), SHAPE, "fewer"), (dict(cache_stride=12804), ALIGN, "16-byte"),
    (dict(k_cache=FAKE + 8), ALIGN, "16-byte"), (dict(work=None), ALIGN, "workspace"),
    (dict(work_bytes=64), WORKSPACE, "needed"), (dict(tree=dict(tokens=8), work_bytes=64), WORKSPACE, "needed"),
    (dict(tree=dict(tokens=8), work=FAKE + 16), WORKSPACE, "workspace"), (dict(tree=dict(pos=None)), ARG, "pos and cells"),
    (dict(tree=dict(cells=None)), ARG, "pos and cells"), (dict(tree=dict(mask=None)), ARG, "trees"),
    (dict(tree=dict(tokens=65537)), ARG, "65536"), (dict(tree=dict(max_nodes=257)), SHAPE, "nodes"),
    (dict(tree=dict(max_count=0)), SHAPE, "max_count")])
def test_layer_refusals(change, code, text):
    tree = _lib.MiTree(**{**TREE, "pos": FAKE, "cells": FAKE, **(change.get("tree") or {})})
    desc = layer_desc(**(change.get("desc") or {}))
    args = {**LAYER, **change, "tree": ctypes.byref(tree), "desc": ctypes.byref(desc)}
    refused(_lib.lib().mi_decoder_layer_tree(*args.values()), code, text)


def test_layer_refuses_no_trees():
    refused(_lib.lib().mi_decoder_layer_tree(*{**LAYER, "desc": ctypes.byref(layer_desc())}.values()), ARG, "trees")
    refused(_lib.lib().mi_decoder_layer_tree(*LAYER.values()), ARG, "descriptor")
    size = _lib.lib().mi_layer_tree_workspace
    tree = _lib.MiTree(**TREE)
    assert size(ctypes.byref(layer_desc()), ctypes.byref(tree)) > 0
    assert size(None, ctypes.byref(tree)) == 0 and size(ctypes.byref(layer_desc()), None) == 0
    assert size(ctypes.byref(layer_desc(head_dim=40)), ctypes.byref(tree)) == 0
    assert size(ctypes.byref(layer_desc()), ctypes.byref(_lib.MiTree(**{**TREE, "tokens": 65537}))) == 0


def test_workspace_of_a_refused_shape_is_zero():
    size = _lib.lib().mi_attend_tree_workspace
    ok = _lib.MiTree(**TREE)
    assert size(8, 2, 64, 0, ctypes.byref(ok)) > 0
    assert size(8, 2, 40, 0, ctypes.byref(ok)) == 0 and size(8, 2, 64, 2, ctypes.byref(ok)) == 0
    assert size(8, 2, 64, 0, None) == 0
    assert size(8, 2, 64, 0, ctypes.byref(_lib.MiTree(**{**TREE, "max_nodes": 300}))) == 0


def test_mojo_structs():
    with open(os.path.join(ROOT, "mojo", "molla_mi.mojo")) as f:
        text = f.read()
    for struct, c in (("QkDesc", _lib.MiQk), ("Tree", _lib.MiTree)):
        part = text[text.index(f"struct {struct}("):]
        assert int(re.search(r"comptime SIZE = (\d+)", part).group(1)) == ctypes.sizeof(c)
        doc = re.search(r'"""(.*?)"""', part, re.S).group(1)
        for name, _ in c._fields_[8 if struct == "QkDesc" else 4:]:
            at = re.search(rf"\b{name}\s+(\d+)", doc)
            assert at and int(at.group(1)) == getattr(c, name).offset, name
