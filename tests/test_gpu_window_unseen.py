"""What a token does not see of a window's cache: finite q8_0 factors of any size, in a
chunk whose tokens lie side by side and in one whose windows leave gaps between them.
(Infinities and NaN: test_gpu_window.py, whose bounds these are too.)"""

import pytest
import torch

from tests.test_gpu_window import Case

pytestmark = pytest.mark.gpu

SIDE_BY_SIDE = [300 + i for i in range(40)]
GAPS = [20, 21, 22, 75, 140, 141, 250, 251, 330, 331, 332, 380]
BACKWARDS = [380, 330, 300, 297, 250, 140, 139, 138, 75, 22, 21, 20]
PADDED = [-1, 300, 301, 302, 303, 304, 305, 306, 307, 360, -1, -1]
# factors of 2^16 - 2^5 and one the other way: the largest there are.  Beside them the
# seen ones, of values to about 4 * 2^-9, lie past the 22 binades that a value's two
# halves hold
LARGE = (0x7bff, -0x0401)


def small(c):
    """c with values small beside the largest factor, and no longer at their rounding."""
    fac = c.v[:, c.kvw // 2:]
    fac.mul_(2.0 ** -9)
    return c


def fill(c, rows, bits):
    for x in (c.k, c.v):
        x.view(torch.int16)[rows, :c.kvw // 2] = 0x7f81  # (129 - 256 and 127)
        x.view(torch.int16)[rows, c.kvw // 2:] = bits


@pytest.mark.parametrize("heads,kvh,d", [(4, 2, 128), (8, 2, 64), (4, 4, 64), (8, 1, 128)])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("pos,window,first", [
    (SIDE_BY_SIDE, 100, 4), (SIDE_BY_SIDE, 1, 0), (SIDE_BY_SIDE, 300, 70), (GAPS, 10, 4), (GAPS, 1, 0), (GAPS, 30, 65),
    (BACKWARDS, 10, 4), (PADDED, 9, 3)])
def test_large_factors_that_no_token_sees(heads, kvh, d, paged, pos, window, first):
    c = small(Case(1, 400, heads, kvh, d, "q8", paged))
    q = torch.randn(len(pos), heads * d, generator=c.g).cuda()
    base = c.run(pos, window, first, True, q=q)
    c.check(base, pos, window, first, True)
    unseen = torch.ones(c.k.shape[0], dtype=torch.bool, device="cuda")
    for t, p in enumerate(pos):
        unseen[c.seen(t, p, window, first, True)] = False
    assert unseen.any()
    for bits in LARGE:
        fill(c, unseen, bits)
        assert torch.equal(c.run(pos, window, first, True, q=q), base)


@pytest.mark.parametrize("kvh,d", [(2, 128), (4, 64)])
def test_large_factors_over_a_long_context(kvh, d):
    """Several splits, slices that are left out between the first positions and the windows."""
    c = small(Case(1, 9000, 8, kvh, d, "q8", True))
    pos = [5000 + i for i in range(70)]
    q = torch.randn(len(pos), 8 * d, generator=c.g).cuda()
    base = c.run(pos, 1000, 100, True, q=q)
    c.check(base, pos, 1000, 100, True, rows=[0, 33, 69])
    unseen = torch.ones(c.k.shape[0], dtype=torch.bool, device="cuda")
    for t, p in enumerate(pos):
        unseen[c.seen(t, p, 1000, 100, True)] = False
    fill(c, unseen, LARGE[0])
    assert torch.equal(c.run(pos, 1000, 100, True, q=q), base)


@pytest.mark.parametrize("d", [64, 128])
def test_large_factors_that_another_token_sees(d):
    """The chunk's other tokens keep their accuracy, by the size of what they see."""
    c = small(Case(1, 400, 4, 2, d, "q8", False))
    pos = [300 + i for i in range(40)]
    fill(c, torch.tensor([270, 320]).cuda(), LARGE[0])
    q = torch.randn(len(pos), 4 * d, generator=c.g).cuda()
    c.k.copy_(Case(1, 400, 4, 2, d, "q8", False).k)  # (finite scores)
    out = c.run(pos, 20, 2, True, q=q)
    blind = [t for t, p in enumerate(pos) if not any(p - 20 < j <= p for j in (270, 320))]
    assert len(blind) > 10
    c.check(out, pos, 20, 2, True, rows=blind)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_with_large_factors_beside(d):
    c = small(Case(6, 400, 4, 2, d, "q8", True))
    pos = [0, 20, 99, 250, 333, 399]
    q = torch.randn(6, 4 * d, generator=c.g).cuda()
    base = c.run(pos, 50, 3, False, q=q)
    c.check(base, pos, 50, 3, False)
    unseen = torch.ones(c.k.shape[0], dtype=torch.bool, device="cuda")
    for t, p in enumerate(pos):
        unseen[c.seen(t, p, 50, 3, False)] = False
    fill(c, unseen, LARGE[0])
    assert torch.equal(c.run(pos, 50, 3, False, q=q), base)
