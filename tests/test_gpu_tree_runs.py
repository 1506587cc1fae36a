"""Tree attention over contexts long enough that a block walks several slices: a
tile is shared by 126 blocks at most, so that one sequence of 20001 positions
gives each block five slices of 32 keys (three of 64).

The gate is 1e-5 of a result's own size, the weighted mean of its values'
magnitudes.  What the kernel may be off by, relative to that: 2^-21 from a weight's
exponent, twice (it is in the sum of weights as well); a score's products, summed
in float32 over 256 dims at most, a few 2^-24 of the sum of their magnitudes, which
these tests keep below 45: some 8 x 45 x 2^-24 / ln 2 at worst, 3e-5, and a tenth of
that where the rounding of a thousand products is not all of one sign; sums
over 160 keys and 126 parts, 2^-24 each step.

Beside it 2^-33 of the largest value there is.  A weight's lower half ends at 2^-36
of the largest weight; over q8_0 it is a weight's product with its factor that ends
there, counted from the largest factor F: a value of at most 127 quants of its own
factor is off by 127 x 2^-36 F, and the largest value is at least 63 F: 2^-34 of it,
averaged over the keys.  Weights below 2^-36 of the largest are zero: below 2^-72 for
the queries here that point at a key (e^-50), times 20001 keys 2^-57.  The matrix cores
align the products of a sum to the largest of their exponents, a zero's counted as
2^-14: 2^-49 of the largest value, for a weight of 2^10 (2^-38 of values up to 2^11,
as measured).
"""

import pytest
import torch

from tests.test_gpu_tree import Step, encode

pytestmark = pytest.mark.gpu

LENGTH = 20001


def results(s):
    """(result, its size) of every token and head in float64."""
    out, size = (torch.zeros(s.tokens, s.heads * s.d, dtype=torch.float64) for _ in range(2))
    k, v, t = s.values(s.k), s.values(s.v), 0
    for b, (n, m) in enumerate(zip(s.lens, s.counts)):
        for _ in range(m):
            rows = s.index[b, torch.tensor(list(range(n)) + [n + i for i in sorted(s.seen[t])])]
            rows = rows[rows >= 0].long()
            for h in range(s.heads):
                at = slice(h // (s.heads // s.kv) * s.d, (h // (s.heads // s.kv) + 1) * s.d)
                o = slice(h * s.d, (h + 1) * s.d)
                p = torch.softmax(k[rows][:, at] @ s.q[t, o].double() * s.scale, 0)
                out[t, o], size[t, o] = p @ v[rows][:, at], p @ v[rows][:, at].abs()
            t += 1
    return out, size


def check_own_size(s, got):
    want, size = results(s)
    gate = 1e-5 * size + 2.0 ** -33 * float(s.values(s.v).abs().max())
    live = sum(s.counts)
    assert torch.isfinite(got[:live]).all()
    off = ((got.double() - want).abs() / gate)[:live]
    assert off.max() <= 1, f"{float(off.max())} of the gate"
    assert (got[live:] == -3.0).all()


def pointed(s, nodes, peak, at, spread=0.02):
    """Queries whose score is `peak` above the others' at position `at`, the others' nearly level."""
    g = torch.Generator().manual_seed(17)
    along = torch.randn(s.d, generator=g)
    keys = spread * torch.randn(len(s.k), s.d, generator=g)
    keys[at] += along * (peak / s.scale) / (along @ along)
    s.k = encode(keys, s.form)
    s.q[:nodes] = along.repeat(s.heads) * (1 + 0.01 * torch.randn(nodes, 1, generator=g))


# with two query heads a key head: up to 16 nodes share their keys among two waves over q8_0
NODES = [(64, 3), (64, 20), (128, 3), (128, 20), (256, 3), (96, 3)]


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", NODES)
@pytest.mark.parametrize("size", [1e-2, 1e-4, 4e-6])
def test_small_values(form, d, nodes, size):
    """One key a query points at, the other keys' weights near 2^-12 of its: each of
    them counts, however small the values are."""
    s = Step(form, [LENGTH], [nodes], 2, 1, d, seed=d)
    pointed(s, nodes, 8.3, 7777)
    g = torch.Generator().manual_seed(18)
    s.v = encode(size * (1 + 0.3 * torch.randn(len(s.v), d, generator=g)), form)
    check_own_size(s, s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", NODES)
@pytest.mark.parametrize("falls", [False, True])
@pytest.mark.parametrize("nodes_only", [False, True])
def test_sizes_that_move_within_a_run(form, d, nodes, falls, nodes_only):
    """Values over 25 octaves in each 300 positions, each 32 dims at a place of their
    own: sums that are not zero when a larger (or smaller) factor comes.  Queries
    that point at a small value are held to its size; with the largest values in the
    nodes alone, the committed ones are held to theirs."""
    s = Step(form, [LENGTH, 45], [nodes, 2], 2, 1, d, seed=d)
    g = torch.Generator().manual_seed(19)
    cells, blocks = len(s.v), d // 32
    place = (torch.arange(cells)[:, None] + 37 * torch.arange(blocks)[None, :]) % 300 / 12.0
    size = 2.0 ** ((25 - place if falls else place) - 15)
    if nodes_only:
        size = torch.where(torch.arange(cells)[:, None] < LENGTH, size * 2.0 ** -8, size)
    s.v = encode((torch.randn(cells, blocks, 32, generator=g) * size[..., None]).reshape(cells, d), form)
    s.k = encode(0.3 * torch.randn(cells, d, generator=g), form)
    check_own_size(s, s.run())
    for at in (3, 7777, 15001, 20000):
        pointed(s, nodes, 60.0, at)
        check_own_size(s, s.run())


@pytest.mark.parametrize("d,nodes", [(64, 3), (64, 40), (128, 3), (128, 70), (256, 3), (96, 3)])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("length", [70, LENGTH])
def test_infinities_that_are_seen(d, nodes, paged, length):
    """An infinite value gives its sign's infinity to whoever sees it, wherever it lies,
    both signs or a NaN give NaN; every other place of the result keeps its bits."""
    s = Step("f16", [length, 40], [nodes, 3], 2, 1, d, seed=d, paged=paged)
    clean = s.run()
    inf, nan = float("inf"), float("nan")
    cells = s.index[0].long()
    for place, v in ((5, inf), (65, -inf), (length // 2 + 1, nan)):  # committed
        s.v[cells[place], place % d] = v
    s.v[cells[2], 7], s.v[cells[length - 3], 7] = inf, -inf
    s.v[cells[3], 9], s.v[cells[length - 1], 9] = -inf, -inf
    s.v[cells[length], 11] = inf  # the first node: itself and its descendants
    s.v[cells[length - 2], 12], s.v[cells[length], 12] = inf, -inf
    want = clean.clone().reshape(s.tokens, 2, d)
    for place, v in ((5, inf), (65, -inf), (length // 2 + 1, nan)):
        want[:nodes, :, place % d] = v
    want[:nodes, :, 7], want[:nodes, :, 9] = nan, -inf
    sees = torch.tensor([0 in s.seen[t] for t in range(nodes)])
    want[:nodes, :, 11] = torch.where(sees[:, None], inf, want[:nodes, :, 11])
    want[:nodes, :, 12] = torch.where(sees[:, None], nan, inf)
    got = s.run().reshape(s.tokens, 2, d)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, 0, 1e38, -1e38), torch.nan_to_num(want, 0, 1e38, -1e38))
