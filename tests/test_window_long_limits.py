"""Workspaces of windowed attention whose bound on the positions is as large as it can
be: a size, not what is left of one past 32 bits."""

import pytest

from molla_amd import _lib

LONG = 2 ** 31 - 1


@pytest.mark.parametrize("head_dim", [32, 96, 512])
@pytest.mark.parametrize("form", [0, 1])
def test_slices_of_the_longest_contexts(head_dim, form):
    ask = lambda window, first, most: _lib.lib().mi_attend_window_workspace(8, 2, head_dim, form, window, first, most, 3, 0)
    below = ask(LONG, 0, LONG - 600)
    assert below > 3 * 8 * 2 ** 25 // 2 * head_dim * 4  # (32 or 64 keys a slice)
    for window, first in ((LONG, 0), (LONG, LONG), (1, LONG), (LONG - 40, 30)):
        assert below <= ask(window, first, LONG) <= below + below // 1000, (window, first)
    assert ask(100, 4, LONG) == ask(100, 4, 100000)
