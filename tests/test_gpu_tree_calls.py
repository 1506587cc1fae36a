"""Calls of a step over trees of drafted tokens that the header allows and the tests
of its results do not make."""

import numpy as np
import pytest
import torch

from molla_amd import gpu
from molla_amd._lib import check, lib
from tests.test_gpu_tree import FORMS, Draft, Step, check_qk, draft, ints, starts_of, words_of

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


@pytest.mark.parametrize("page", [1, 4, 16])
def test_pages_of_rejected_drafts_go_back(page):
    """Steps of which a part is taken back, in the header's way and without a look from
    the host: no page is lost, none is held twice, and kept positions keep their cells."""
    batch, width, new, pages = 5, 24 if page > 1 else 130, 9, 5 * 130 // page
    g = torch.Generator().manual_seed(page)
    ctx = gpu.DeviceContext(0)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    free = torch.cat([torch.randperm(pages, generator=g), torch.zeros(1, dtype=torch.int64)]).to(torch.int32).cuda()
    count, left, lengths = ints([pages]), ints([0, 0]), ints([0] * batch)
    index = torch.full((batch, width * page), -1, dtype=torch.int32, device="cuda")
    starts, cells = ints([0] * (batch + 1)), ints([-1] * (batch * new))
    col = torch.arange(width, device="cuda")
    held_cells = [[] for _ in range(batch)]
    for step in range(20):
        news = torch.randint(0, new + 1, (batch,), generator=g).to(torch.int32).cuda()
        kept = torch.minimum(torch.randint(0, 6, (batch,), generator=g).to(torch.int32).cuda(), news)
        gpu.device_page_plan(ctx, page, lengths, news, table, free[:pages], count, left, starts, None, None, cells, index)
        # the pages behind the kept positions go back: a place on the list each, the others to the spare slot
        keep, had = -(-(lengths + kept) // page), -(-(lengths + news) // page)
        back = ((col >= keep[:, None]) & (col < had[:, None])).flatten()
        place = torch.where(back, left[0] + torch.cumsum(back, 0) - 1, pages)
        free.index_put_((place,), table.flatten())
        count.copy_(left[:1] + back.sum())
        lengths += kept
        ctx.synchronize()
        assert left[1] == 0
        on_list = free[:int(count)].tolist()
        in_use = [table[b, c].item() for b in range(batch) for c in range(-(-int(lengths[b]) // page))]
        assert sorted(on_list + in_use) == list(range(pages)), step
        for b in range(batch):
            n = int(lengths[b])
            assert index[b, :len(held_cells[b])].tolist() == held_cells[b]
            held_cells[b] = index[b, :n].tolist()
            assert min(held_cells[b], default=0) >= 0


def test_qk_outputs_between_rows():
    """Outputs at one stride with the inputs, in what those leave free, and in place: as outputs apart."""
    heads, kv, d, tokens = 8, 2, 64, 50
    qw, kvw = heads * d, kv * d
    g = torch.Generator().manual_seed(2)
    steps = torch.from_numpy(gpu.rope_steps(d, 10000.0)).cuda()
    data = torch.randn(tokens, qw + 2 * kvw, generator=g).cuda()
    ctx, outs = gpu.DeviceContext(0), []
    for how in ("apart", "between", "in place"):
        row = torch.zeros(tokens, 2 * qw + 3 * kvw, device="cuda")
        # q | q_out | k | k_out | v
        q, q_out, k, k_out, v = torch.split(row, [qw, qw, kvw, kvw, kvw], 1)
        if how == "apart":
            q_out, k_out = torch.zeros(tokens, qw, device="cuda"), torch.zeros(tokens, kvw, device="cuda")
        elif how == "in place":
            q_out, k_out = q, k
        q.copy_(data[:, :qw]), k.copy_(data[:, qw:qw + kvw]), v.copy_(data[:, qw + kvw:])
        kc, vc = (torch.zeros(tokens, kvw, dtype=torch.float16, device="cuda") for _ in range(2))
        gpu.device_qk_norm_rope(ctx, q, k, v, heads, kv, d, d, True, steps, ints(range(tokens)), q_out, kc, vc,
                                ints(range(tokens)), k_out=k_out)
        ctx.synchronize()
        outs.append([t.clone() for t in (q_out, k_out, kc, vc, v)])
    for other in outs[1:]:
        for a, b in zip(outs[0], other):
            assert torch.equal(a, b)


def test_tree_plan_in_the_place_of_parents():
    """pos, or a mask of one word, where the parents were."""
    ctx = gpu.DeviceContext(0)
    counts, lens = [20, 0, 31], [5, 6, 7]
    parents, seen, depth = draft(counts, 3)
    words = words_of(seen, 1)
    first = np.repeat(lens, counts)
    for which in ("pos", "mask"):
        p, other = ints(parents), ints([0] * len(parents))
        pos, mask = (p, other) if which == "pos" else (other, p)
        gpu.device_tree_plan(ctx, starts_of(counts), ints(lens), p, 31, pos, mask)
        ctx.synchronize()
        assert pos.tolist() == [int(n) + d for n, d in zip(first, depth)]
        assert mask.tolist() == words[:, 0].tolist()


def test_page_plan_of_one_position_a_page():
    """With pages of one position the table and the list are one buffer."""
    lens, news, width = [3, 0, 7], [4, 5, 0], 12
    free = torch.randperm(40).to(torch.int32)[:20]
    table = torch.full((3, width), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        table[b, :n] = torch.arange(n) + 50 + 10 * b
    outs = []
    for shared in (False, True):
        t = table.cuda()
        index = t if shared else table.cuda()
        starts, cells, left = ints([0] * 4), ints([-1] * 9), ints([0, 0])
        gpu.device_page_plan(gpu.DeviceContext(0), 1, ints(lens), ints(news), t, free.cuda(), ints([20]), left, starts, None,
                             None, cells, index)
        torch.cuda.synchronize()
        outs.append((t, index, starts, cells, left))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


# ---- launches of more than 2^32 threads ------------------------------------------
@pytest.mark.parametrize("d", [32, 64])
def test_qk_of_many_tokens(d):
    """More than 2^26 rows: each as in a short call."""
    tokens, ctx = (1 << 26) + 9, gpu.DeviceContext(0)
    g = torch.Generator(device="cuda")
    g.manual_seed(d)
    q = torch.randn(tokens, d, generator=g, device="cuda")
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    steps = torch.from_numpy(gpu.rope_steps(d, 10000.0)).cuda()
    out = torch.full((tokens, d), -3.0, device="cuda")
    gpu.device_qk_norm_rope(ctx, q, q, None, 1, 1, d, d, True, steps, pos, out)
    for first in (0, tokens // 2, tokens - 1000):
        part = torch.full((1000, d), -4.0, device="cuda")
        at = slice(first, first + 1000)
        gpu.device_qk_norm_rope(ctx, q[at], q[at], None, 1, 1, d, d, True, steps, pos[at], part)
        ctx.synchronize()
        assert torch.equal(out[at], part)
    assert not bool((out == -3.0).all(1).any())


def test_tree_plan_of_many_sequences():
    batch, ctx = (1 << 24) + 5, gpu.DeviceContext(0)
    counts = torch.zeros(batch, dtype=torch.int32)
    live = [0, 77, 1 << 23, batch - 2, batch - 1]
    sizes = [256, 3, 40, 1, 100]
    for b, n in zip(live, sizes):
        counts[b] = n
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)]).to(torch.int32).cuda()
    lengths = torch.arange(batch, dtype=torch.int32).cuda()
    parents, seen, depth = draft(sizes, 6)
    pos, mask = ints([-3] * len(parents)), ints([[-3] * 8] * len(parents))
    gpu.device_tree_plan(ctx, starts, lengths, ints(parents), 256, pos, mask)
    ctx.synchronize()
    assert pos.tolist() == [int(n) + d for n, d in zip(np.repeat(live, sizes), depth)]
    assert (mask.cpu().numpy() == words_of(seen, 8)).all()


@pytest.mark.parametrize("heads,kv,d,batch", [(8, 1, 256, 40000), (8, 1, 64, 131100), (8, 1, 128, 65600), (8, 2, 96, 40000)])
def test_attend_of_many_sequences(heads, kv, d, batch):
    """Room for more rows than a launch has threads; the rows that are there are shared by blocks."""
    s = Step("f16", [300, 41, 290, 7], [5, 0, 9, 2], heads, kv, d, seed=1, paged=True)
    live = [0, 500, batch - 2, batch - 1]
    lens, counts = torch.zeros(batch, dtype=torch.int32), torch.zeros(batch, dtype=torch.int64)
    index = torch.full((batch, s.room), -1, dtype=torch.int32)
    for i, b in enumerate(live):
        lens[b], counts[b], index[b] = s.lens[i], s.counts[i], s.index[i]
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)]).to(torch.int32)
    mask = np.concatenate([words_of(s.seen, 8), np.full((s.tokens - len(s.seen), 8), -1, np.int32)])
    out = torch.full((s.tokens, heads * d), -3.0, device="cuda")
    ctx = gpu.DeviceContext(0)
    gpu.device_attend_tree(ctx, s.q.cuda(), s.k.cuda(), s.v.cuda(), heads, kv, d, s.scale, starts.cuda(), lens.cuda(), ints(mask),
                           256, s.max_count, out, kv_index=index.cuda())
    ctx.synchronize()
    s.check(out.cpu())


# ---- captured calls --------------------------------------------------------------
@pytest.mark.parametrize("form,heads,kv,d", [("f16", 4, 2, 256), ("q8", 4, 2, 96)])
def test_a_first_call_that_is_captured(form, heads, kv, d):
    """A context whose first calls are a capture, its workspace made there: each replay as
    the eager calls between them, and the workspace outlives the graph."""
    stream = torch.cuda.Stream()
    ctx = gpu.DeviceContext(0, stream)
    s = Draft(ctx, form, heads, kv, d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        s.step()
    for _ in range(3):
        s.out.fill_(-3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        replayed = s.check()
        s.out.fill_(-3.0)
        torch.cuda.synchronize()
        s.step()
        ctx.synchronize()
        assert torch.equal(s.out, replayed)
    del graph
    other = torch.full((1 << 22,), 7.0, device="cuda")
    s.out.fill_(-3.0)
    torch.cuda.synchronize()
    s.step()
    ctx.synchronize()
    assert torch.equal(s.out, replayed) and bool((other == 7.0).all())


def test_two_graphs_of_one_context():
    """Captured on one context they share its workspace, and run one after the other."""
    stream = torch.cuda.Stream()
    ctx = gpu.DeviceContext(0, stream)
    steps, graphs, want = [Draft(ctx, "f16"), Draft(ctx, "q8", 8, 8, 128)], [], []
    torch.cuda.synchronize()
    for s in steps:
        s.step()
        ctx.synchronize()
        want.append(s.check())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            s.step()
    for order in ((0, 1, 0), (1, 1, 0, 1)):
        for s in steps:
            s.out.fill_(-3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for i in order:
                graphs[i].replay()
        ctx.synchronize()
        for s, w in zip(steps, want):
            assert torch.equal(s.out, w)


# ---- the widths and sizes between the others' ---------------------------------------
@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d", [160, 192, 224, 288, 320, 352, 384, 416, 448, 480])
def test_every_head_width(form, d):
    """Attention, then norm, rotation and store, at the widths that no other test has."""
    for paged, heads, kv in ((False, 2, 1), (True, 4, 1)):
        s = Step(form, [70, 0, 41], [5, 3, 0], heads, kv, d, seed=d, paged=paged)
        s.check(s.run())
    check_qk(5, 4, 1, d, d, True, True, False, form)
    check_qk(6, 2, 2, d, d // 2, False, True, True, form, pad=0)
    check_qk(3, 1, 1, d, 2, True, False, False, form, pad=4, in_place=True)


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d", [256, 512, 32])
def test_eight_query_heads_a_key_head(form, d):
    s = Step(form, [50, 300], [33, 2], 16, 2, d, seed=d, paged=True)
    s.check(s.run())


def test_tree_plan_without_positions():
    ctx = gpu.DeviceContext(0)
    parents, seen, _ = draft([9, 2], 1)
    mask = ints([[-3]] * 12)
    gpu.device_tree_plan(ctx, starts_of([9, 2]), ints([4, 5]), ints(parents + [0]), 9, None, mask)
    ctx.synchronize()
    assert (mask.cpu().numpy()[:11] == words_of(seen, 1)).all() and int(mask[11]) == -3


def test_page_plan_of_an_empty_free_list():
    """A list of no pages lies nowhere, whatever its address."""
    starts, cells, left, table = ints([0] * 3), ints([-3] * 4), ints([0, 0]), ints([[7, -1], [3, -1]])
    lens, news, none = ints([5, 15]), ints([1, 3]), ints([0])
    check(lib().mi_page_plan(None, 2, 16, lens.data_ptr(), news.data_ptr(), table.data_ptr(), 2, cells.data_ptr() + 8, 0,
                             none.data_ptr(), left.data_ptr(), None, 0, 4, starts.data_ptr(), None, None, cells.data_ptr()))
    torch.cuda.synchronize()
    assert cells.tolist() == [7 * 16 + 5, 3 * 16 + 15, -1, -1] and left.tolist() == [0, 1]


def test_rows_that_start_behind_the_first():
    """starts[0] may be past 0: the rows ahead of it keep what they held."""
    s = Step("f16", [40, 33], [5, 6], 4, 2, 64, spare=7)
    want, ctx = s.run(), gpu.DeviceContext(0)
    e = s.dev
    q, mask = torch.roll(e["q"], 4, 0), torch.roll(e["mask"], 4, 0)
    out = torch.full_like(q, -3.0)
    gpu.device_attend_tree(ctx, q, e["k"], e["v"], 4, 2, 64, s.scale, e["starts"] + 4, e["lengths"], mask, s.max_nodes,
                           s.max_count, out, cache_stride=s.room * s.k.shape[1])
    ctx.synchronize()
    assert torch.equal(out.cpu()[4:15], want[:11]) and bool((out[:4] == -3.0).all()) and bool((out[15:] == -3.0).all())
