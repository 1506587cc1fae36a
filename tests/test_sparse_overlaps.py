"""Outputs and workspaces that share a byte with the weights or the caches a call reads
are refused (on the host: nothing is launched, the pointers are made up)."""

import ctypes

import pytest

from molla_amd import _lib
from tests.test_sparse_refusals import ARG, WORK, experts, far, matmul, mlp, refused
from tests.test_window_overlaps import far as apart, window

GATE, DOWN = 2048 * 144, 1024 * 288  # bytes of the stacks of experts()


def room(tokens=3, used=2):
    return _lib.lib().mi_experts_workspace(ctypes.byref(experts()), tokens, used)


@pytest.mark.parametrize("at,size", [(1, GATE), (2, GATE), (3, DOWN)])
def test_mlp(at, size):
    out, work = 3 * 256 * 4, room()
    for p in (far(at), far(at) + 1024, far(at) + size - 16, far(at) - out + 16):
        refused(mlp(out=p), ARG, "lies in")
    for p in (far(at), far(at) + size - 256, far(at) - work + 256):
        refused(mlp(work=p), ARG, "workspace lies")
    for p in (far(at) + size, far(at) - out):  # (they only touch: on to the workspace's size)
        refused(mlp(out=p, bytes=0), WORK, "workspace of 0")


def test_matmul():
    size = 4 * 64 * 144
    need = _lib.lib().mi_experts_matmul_workspace(4, 256, 2, 8)
    for p in (far(1), far(1) + size - 256, far(1) - need + 256):
        refused(matmul(work=p), ARG, "workspace lies")


ROW = 256  # halves of a cached position, 2 heads of 128 in f16


@pytest.mark.parametrize("cache", ["k", "v"])
@pytest.mark.parametrize("stride", [0, 500 * ROW, 1 << 20])
def test_window_caches(cache, stride):
    end = 2 * (2 * stride + 500 * ROW)  # bytes of three sequences, or of one
    at = {"k": apart(2), "v": apart(3)}[cache]
    for p in (at, at + end - 16, at - 3 * 4096 + 16):
        rc, words = window(index=None, cache_stride=stride, out=p)
        assert rc == ARG and " lies in " in words, (rc, words)
    for p in (at, at + (end - 1) // 256 * 256, at - 256):
        rc, words = window(index=None, cache_stride=stride, work=p)
        assert rc == ARG and " lies in " in words, (rc, words)
    rc, words = window(index=None, cache_stride=stride, out=at + end, bytes=0)
    assert rc == WORK, (rc, words)


def test_between_the_caches_of_two_sequences():
    """What lies between them may be anything else's."""
    s, run = 2 << 20, 2 * 500 * ROW  # bytes from one to the next, and of one
    for t in range(3):
        at = apart(2) + t * s
        rc, words = window(index=None, cache_stride=1 << 20, out=at + run, bytes=0)
        assert rc == WORK, (t, rc, words)
        rc, words = window(index=None, cache_stride=1 << 20, out=at - 3 * 4096, bytes=0)
        assert rc == WORK, (t, rc, words)
        for p in (at + run - 16, at - 3 * 4096 + 16, at + 4096):
            rc, words = window(index=None, cache_stride=1 << 20, out=p)
            assert rc == ARG and " lies in " in words, (t, rc, words)
        rc, words = window(index=None, cache_stride=1 << 20, work=at + run + 256 & ~255, bytes=0)
        assert rc == WORK, (t, rc, words)


def test_window_of_one_token():
    """One token's cache is one sequence, whatever the stride."""
    rc, words = window(index=None, cache_stride=1 << 20, tokens=1, out=apart(2) + 2 * 500 * ROW, bytes=0)
    assert rc == WORK, (rc, words)
    rc, words = window(index=None, cache_stride=1 << 20, tokens=1, out=apart(2) + 2 * 500 * ROW - 16)
    assert rc == ARG, (rc, words)


@pytest.mark.parametrize("form,row", [(0, 256), (1, 136)])
def test_window_forms(form, row):
    rc, words = window(index=None, form=form, out=apart(3) + 2 * 500 * row - 16)
    assert rc == ARG and " lies in " in words, (rc, words)
    rc, words = window(index=None, form=form, out=apart(3) + 2 * 500 * row, bytes=0)
    assert rc == WORK, (rc, words)
