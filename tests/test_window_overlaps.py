"""mi_attend_window refuses an output or a workspace that lies in another buffer
(on the host: nothing is launched, the pointers are made up)."""

import pytest

from molla_amd import _lib

ARG, WORK = -1, -5


def far(n):
    return n << 40


def window(**kw):
    a = dict(form=0, q=far(1), q_stride=1024, k=far(2), v=far(3), cache_stride=0, index=far(7), index_stride=600, heads=8,
             kv_heads=2, head_dim=128, scale=0.1, window=100, first=4, pos=far(4), max_count=500, tokens=3, out=far(5),
             work=far(6), bytes=1 << 30)
    a.update(kw)
    rc = _lib.lib().mi_attend_window(None, *a.values())
    return rc, _lib.lib().mi_last_error().decode()


LISTS = 4 * (2 * 600 + 500)  # bytes of three lists, 600 apart


@pytest.mark.parametrize("kw", [
    dict(out=far(4)), dict(pos=far(5) + 3 * 4096 - 4), dict(out=far(7)), dict(out=far(7) + LISTS - 16),
    dict(work=far(1)), dict(work=far(1) + 2 * 4096 + 3840), dict(work=far(4)), dict(work=far(7) + 6656),
    dict(work=far(5)), dict(work=far(5) + 2 * 4096 + 3840), dict(out=far(6) + 1024), dict(pos=far(6) + 512),
    dict(index=far(6) - LISTS + 4)])
def test_refused(kw):
    rc, words = window(**kw)
    assert rc == ARG and " lies in " in words, (rc, words)


@pytest.mark.parametrize("kw", [
    dict(pos=far(5) + 3 * 4096), dict(pos=far(5) - 12), dict(index=far(5) - LISTS), dict(index=far(6) - LISTS),
    dict(index=far(6) - 2000, index_stride=0), dict(work=far(1) + 3 * 4096), dict(work=far(5) + 3 * 4096)])
def test_buffers_that_only_touch_pass(kw):
    """The workspace's size is what is looked at behind the overlaps."""
    rc, words = window(bytes=0, **kw)
    assert rc != ARG and "workspace of 0 bytes" in words, (rc, words)
