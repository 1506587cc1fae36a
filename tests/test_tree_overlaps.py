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


def plan():
    """Four requests, tables of 8 pages of 16, a list of 10 free pages, 32 token rows; every buffer 0x1000 bytes on."""
    at = {n: FAKE + 0x1000 * i for i, n in enumerate(("lengths", "news", "table", "free_pages", "free_count", "free_left",
                                                      "kv_index", "starts", "seq", "pos", "cells"))}
    a = dict(stream=None, batch=4, page=16, lengths=0, news=0, table=0, table_stride=8, free_pages=0, free_size=10,
             free_count=0, free_left=0, kv_index=0, index_stride=128, max_tokens=32, starts=0, seq=0, pos=0, cells=0)
    a.update(at)
    return at, a


SIZES = dict(lengths=4, news=4, table=32, free_pages=10, free_count=1, free_left=2, kv_index=512, starts=5, seq=32, pos=32, cells=32)


@pytest.mark.parametrize("written", ["starts", "free_left", "seq", "pos", "cells", "kv_index", "table"])
@pytest.mark.parametrize("read", ["lengths", "news", "free_pages", "free_count", "table"])
@pytest.mark.parametrize("last", [False, True])
def test_page_plan_outputs_among_inputs(written, read, last):
    if written == read:
        return
    at, a = plan()
    # the first value of one at the last of the other
    a[written] = at[read] + (4 * (SIZES[read] - 1) if last else -4 * (SIZES[written] - 1))
    if (written, read) == ("free_left", "free_count"):
        text = "free_left may not be free_count"
    else:
        text = f"{'the table' if written == 'table' else written} lies in {'the table' if read == 'table' else read}"
    refused(_lib.lib().mi_page_plan(*a.values()), ARG, text)


def test_page_plan_list_in_the_table():
    _, a = plan()
    a["kv_index"] = a["table"]
    refused(_lib.lib().mi_page_plan(*a.values()), ARG, "kv_index lies in the table")
    refused(_lib.lib().mi_page_plan(*{**a, "page": 1}.values()), ARG, "kv_index lies in the table")  # (at another stride)


@pytest.mark.parametrize("change,text", [
    (dict(pos=FAKE), "pos lies in starts"), (dict(pos=FAKE + 8), "pos lies in starts"), (dict(pos=FAKE - 60), "pos lies in starts"),
    (dict(mask=FAKE), "mask lies in starts"), (dict(pos=FAKE + 0x1004), "pos lies in lengths"),
    (dict(mask=FAKE + 0x1004), "mask lies in lengths"), (dict(pos=FAKE + 0x2004), "pos lies in parents"),
    (dict(mask=FAKE + 0x2004), "mask lies in parents"), (dict(mask=FAKE + 0x2000, max_nodes=40), "mask lies in parents"),
    (dict(pos=FAKE + 0x4000), "pos lies in the mask"), (dict(pos=FAKE + 0x4000 + 60), "pos lies in the mask"),
    (dict(pos=FAKE + 0x2000, mask=FAKE + 0x2000), "pos lies in the mask")])
def test_tree_plan_outputs_among_inputs(change, text):
    a = dict(stream=None, batch=2, starts=FAKE, lengths=FAKE + 0x1000, parents=FAKE + 0x2000, max_nodes=8, tokens=16,
             pos=FAKE + 0x3000, mask=FAKE + 0x4000)
    refused(_lib.lib().mi_tree_plan(*{**a, **change}.values()), ARG, text)
