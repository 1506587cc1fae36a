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


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", NODES + [(128, 70), (32, 3), (512, 3)])
@pytest.mark.parametrize("rise", [0.004, 0.08, 1.9, 2.76, 2.85, 5.6, -0.08])
def test_rising_scores_within_a_run(form, d, nodes, rise):
    """Scores that rise over each 450 positions, by `rise` a key or (from 1 on) a 50th
    key: the running maximum moves inside a block's run at every slice, at some, or by
    just less and just more than what the sums are left alone for."""
    s = Step(form, [LENGTH, 40], [nodes, 2], 1, 1, d)
    g = torch.Generator().manual_seed(7)
    along = torch.randn(d, generator=g)
    steps = torch.arange(LENGTH, dtype=torch.float32) % 450
    score = rise * (steps if rise < 1 else (steps / 50).floor())
    s.k[:LENGTH] = encode((score - (score.max() + score.min()) / 2)[:, None] / s.scale * along / (along @ along) +
                          0.02 * torch.randn(LENGTH, d, generator=g), form)
    s.q[:nodes] = along * (1 + 0.01 * torch.randn(nodes, 1, generator=g))
    check_own_size(s, s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", NODES + [(128, 70), (32, 20), (512, 3)])
def test_positions_not_held_within_a_run(form, d, nodes):
    """Cells that are not held: one in seven, whole slices, the ends of some, all of a sequence's."""
    s = Step(form, [LENGTH, 300, 90], [nodes, 3, 2], 2, 1, d, seed=d, paged=True)
    s.index[0, 5:LENGTH - 900:7] = -1
    for a, n in ((0, 32), (640, 64), (3000, 1000), (8000 - 3, 70), (LENGTH - 500, 40), (LENGTH - 2, 1)):
        s.index[0, a:a + n] = -1
    s.index[1, 40:200] = -1
    s.index[2, :90] = -1
    check_own_size(s, s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("heads,kv,d,nodes", [(4, 2, 96, 6), (4, 4, 32, 20), (2, 1, 512, 5), (4, 2, 64, 6), (2, 1, 128, 40),
                                              (2, 1, 256, 6)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -65504.0])
@pytest.mark.parametrize("length,paged", [(70, False), (70, True), (LENGTH, True)])
def test_what_is_not_seen(form, heads, kv, d, nodes, bad, length, paged):
    """What lies in nodes that a token does not see, in slots behind the sequence and in
    cells that are not held changes no bit of its result, at every kind of head width
    and where a block walks several slices."""
    s = Step(form, [length, 30], [nodes, nodes], heads, kv, d, seed=d, paged=paged)
    for t in range(2 * nodes):  # the last node is seen by itself alone, the one before by nobody
        s.seen[t] -= {nodes - 2}
        if t % nodes != nodes - 1:
            s.seen[t] -= {nodes - 1}
    if paged:
        s.index[0, 11::23] = -1
        s.index[1, 0] = -1
    clean = s.run()
    check_own_size(s, clean)
    kvw = kv * d
    held = {int(s.index[b, j]) for b, n in enumerate(s.lens) for j in range(n + nodes) if j != n + nodes - 2}
    hidden = torch.tensor([i for i in range(len(s.k)) if i not in held])
    for c in (s.k, s.v):
        if form == "f16":
            c[hidden] = bad
        else:
            c[hidden, kvw // 2:kvw // 2 + kvw // 32] = bad
    assert torch.equal(s.run(), clean)
    # the last node's own value (not its key) goes to itself alone
    for b, n in enumerate(s.lens):
        i = int(s.index[b, n + nodes - 1])
        if form == "f16":
            s.v[i] = bad
        else:
            s.v[i, kvw // 2:kvw // 2 + kvw // 32] = bad
    got = s.run()
    last = [nodes - 1, 2 * nodes - 1]
    others = [t for t in range(s.tokens) if t not in last]
    assert torch.equal(got[others], clean[others])
    if not abs(bad) < float("inf"):
        assert not torch.isfinite(got[last]).any()
