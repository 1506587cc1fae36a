"""Calls of a step over trees of drafted tokens that the header allows and the tests
of its results do not make."""

import pytest
import torch

from molla_amd import gpu
from tests.test_gpu_tree import FORMS, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,pad", [(64, 0), (128, 4), (96, 0)])
def test_cells_that_two_tokens_name(form, d, pad):
    """Their row is nobody's; every other row and the rotated heads are as without them."""
    heads, kv, tokens, rows = 8, 4, 40, 64
    g = torch.Generator().manual_seed(d)
    row = torch.randn(tokens, (heads + 2 * kv) * d + pad, generator=g).cuda()
    steps = torch.from_numpy(gpu.rope_steps(d, 10000.0)).cuda()
    cells = torch.randperm(rows, generator=g)[:tokens].to(torch.int32)
    twice = cells.clone()
    twice[7], twice[30], twice[31] = cells[3], cells[12], cells[12]
    ctx, outs = gpu.DeviceContext(0), []
    for c in (cells, twice):
        q, k = torch.zeros(tokens, heads * d, device="cuda"), torch.zeros(tokens, kv * d, device="cuda")
        kc, vc = (torch.zeros(rows, gpu.cache_row(FORMS[form], kv * d), dtype=torch.float16, device="cuda") for _ in range(2))
        gpu.device_qk_norm_rope(ctx, row[:, :heads * d], row[:, heads * d:(heads + kv) * d],
                                row[:, (heads + kv) * d:(heads + 2 * kv) * d], heads, kv, d, d, True, steps,
                                ints(range(tokens)), q, kc, vc, c.cuda(), FORMS[form], k_out=k)
        ctx.synchronize()
        outs.append((q, k, kc, vc))
    for a, b in zip(outs[0][:2], outs[1][:2]):
        assert torch.equal(a, b)
    own = [int(cells[t]) for t in range(tokens) if t not in (3, 7, 12, 30, 31)]
    unnamed = [i for i in range(rows) if i not in cells.tolist()] + [int(cells[t]) for t in (7, 30, 31)]
    for a, b in zip(outs[0][2:], outs[1][2:]):
        assert torch.equal(a[own].view(torch.int16), b[own].view(torch.int16)) and (b[unnamed] == 0).all()


@pytest.mark.parametrize("batch", [3, 300])
def test_page_plan_of_the_most_token_rows(batch):
    """Requests that want 2^30 rows each, of 2^30 rows (4 GiB): the sum of two passes 31 bits."""
    rows, ctx = 1 << 30, gpu.DeviceContext(0)
    news = [rows, rows, 5] + [rows] * (batch - 3)
    table = torch.arange(4 * batch, dtype=torch.int32, device="cuda").reshape(batch, 4)
    starts, cells, left = ints([-9] * (batch + 1)), torch.full((rows,), -3, dtype=torch.int32, device="cuda"), ints([-5, -5])
    for first in (0, 7):  # (7: the second request's sum is cut inside it)
        gpu.device_page_plan(ctx, 16, ints([64] * batch), ints([rows - first] + news[1:]), table, ints([1]), ints([0]), left,
                             starts, None, None, cells)
        ctx.synchronize()
        assert starts.tolist() == [0, rows - first] + [rows] * (batch - 1) and left.tolist() == [0, 0]
        assert bool((cells == -1).all())  # (the table has no room behind the 64 positions)
    gpu.device_page_plan(ctx, 16, ints([60] * batch), ints(news), table, ints([1]), ints([0]), left, starts, None, None, cells)
    ctx.synchronize()
    assert starts.tolist() == [0] + [rows] * batch
    assert cells[:4].tolist() == [60, 61, 62, 63] and bool((cells[4:] == -1).all())
