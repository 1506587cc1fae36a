"""A value that is not finite makes its place of a windowed token's result not finite,
also where its key's weight is zero beside the largest score: in the share or slice of
that score, in another one, in a chunk."""

import pytest
import torch

from tests.test_gpu_window import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kvh,d", [(4, 2, 64), (4, 2, 128), (8, 1, 128), (2, 1, 256), (4, 2, 96), (2, 1, 32)])
@pytest.mark.parametrize("n,chunk", [(1, False), (3, False), (2, True), (12, True)])
@pytest.mark.parametrize("paged", [False, True])
def test_weights_of_zero(heads, kvh, d, n, chunk, paged):
    room, window, first = 5000, 4000, 5
    seqs = 1 if chunk else n
    c = Case(seqs, room, heads, kvh, d, "f16", paged)
    c.scale = 1.0
    pos = [4600 + i for i in range(n)]
    q = torch.randn(n, heads * d, generator=c.g).cuda()
    q[:, ::d] = 30.0
    cell = lambda s, j: c.index[s, j].long() if paged else s * room + j
    for s in range(seqs):
        for j in range(4590, 4600):  # scores of 900 there, beside about 0 +- 16 and 30 at dim 0
            c.k[cell(s, j), ::d] = 30.0
    base = c.run(pos, window, first, chunk, q=q).view(n, kvh, heads // kvh, d)
    assert torch.isfinite(base).all()
    bad = {1: (0, 3), 4: (kvh - 1, 7), 700: (0, 12), 1500: (0, 30), 2233: (kvh - 1, 20), 3100: (0, d - 1), 4400: (0, 25),
           4594: (0, 9)}
    places = torch.zeros(kvh, d, dtype=torch.bool, device="cuda")
    for i, (j, (h, at)) in enumerate(bad.items()):
        for s in range(seqs):
            c.v[cell(s, j), h * d + at] = (float("inf"), float("-inf"), float("nan"))[i % 3]
        places[h, at] = True
    out = c.run(pos, window, first, chunk, q=q).view(n, kvh, heads // kvh, d)
    hit = places[None, :, None].expand_as(out)
    assert not torch.isfinite(out[hit]).any()
    assert torch.isfinite(out[~hit]).all()
