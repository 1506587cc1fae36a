"""A step over trees of drafted tokens: the page plan, the tree plan, the
per-head norm with rotation and cache store, and the trees' attention, each
against a plain implementation (whole numbers by loops, the rest in float64),
then the four in a row.

Attention's gate is that of the other attention tests, 1e-5 of the largest value
a row can average (scores here are a few units: a product of 128 values summed in
float32 is off by about sqrt(128) 2^-24 of the largest partial sum, some 3e-6 in a
weight's exponent).
"""

import numpy as np
import pytest
import torch

from molla_amd import gpu

pytestmark = pytest.mark.gpu

FORMS = {"f16": gpu.CACHE_F16, "q8": gpu.CACHE_Q8}


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def starts_of(counts):
    return ints(np.concatenate([[0], np.cumsum(counts)]))


def draft(counts, seed, kind="random"):
    """parents of trees of these sizes, and (set of nodes seen, depth) of each token, by loops"""
    rng = np.random.default_rng(seed)
    parents, seen, depth = [], [], []
    for n in counts:
        p, s, d = [], [], []
        for i in range(n):
            if kind == "chain":
                up = i - 1
            elif kind == "roots":
                up = -1
            else:
                up = int(rng.integers(max(-1, i - 5), i)) if i else -1
            p.append(up)
            s.append({i} | (s[up] if up >= 0 else set()))
            d.append(d[up] + 1 if up >= 0 else 0)
        parents += p
        seen += s
        depth += d
    return parents, seen, depth


def words_of(seen, words):
    out = np.zeros((len(seen), words), np.uint32)
    for t, s in enumerate(seen):
        for i in s:
            out[t, i // 32] |= np.uint32(1 << (i % 32))
    return out.view(np.int32)


# ---- the page plan ------------------------------------------------------------
def plan_by_loops(page, lens, news, table, free, n_free, index, tokens):
    """the header's words, one position at a time"""
    table, index = table.copy(), None if index is None else index.copy()
    starts, seq, pos, cells = [0], [], [], []
    room = table.shape[1] * page
    if index is not None:
        room = min(room, index.shape[1])
    n_free = left = min(max(n_free, 0), len(free))
    want = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        n, m = max(n, 0), max(m, 0)
        m = min(m, tokens - len(cells))
        for j in range(n, n + m):
            cell = -1
            if j < room:
                if j % page == 0:
                    want += 1
                    table[b, j // page] = free[n_free - want] if want <= n_free else -1
                at = int(table[b, j // page])
                cell = at * page + j % page if at >= 0 and at * page + j % page < 2 ** 31 else -1
                if index is not None:
                    index[b, j] = cell
            seq.append(b)
            pos.append(min(j, 2 ** 31 - 1))
            cells.append(cell)
        starts.append(len(cells))
    return starts, seq, pos, cells, table, index, [max(left - want, 0), max(want - left, 0)]


def check_plan(page, lens, news, width, n_free, free_size, tokens, with_index=True, index_stride=None, seed=0, stream=None):
    rng = np.random.default_rng(seed)
    b = len(lens)
    have = [min(-(-max(n, 0) // page), width) for n in lens]
    pages = rng.permutation(sum(have) + free_size + 3).astype(np.int32)
    table = np.full((b, width), -7, np.int32)
    at = 0
    for i, h in enumerate(have):
        table[i, :h] = pages[at:at + h]
        at += h
    free = pages[at:at + free_size]
    index = rng.integers(-1, 50, (b, index_stride or width * page)).astype(np.int32) if with_index else None
    want = plan_by_loops(page, lens, news, table, free, n_free, index, tokens)
    ctx = gpu.DeviceContext(0, stream)
    d = dict(lengths=ints(lens), news=ints(news), table=ints(table), free_pages=ints(free), free_count=ints([n_free]),
             free_left=ints([-5, -5]), starts=ints([-9] * (b + 1)), seq=ints([-3] * tokens), pos=ints([-3] * tokens),
             cells=ints([-3] * tokens), kv_index=None if index is None else ints(index))
    torch.cuda.synchronize()
    gpu.device_page_plan(ctx, page, **d)
    ctx.synchronize()
    starts, seq, pos, cells, table, index, left = want
    total = len(cells)
    assert d["starts"].tolist() == starts
    for name, w in (("seq", seq), ("pos", pos), ("cells", cells)):
        got = d[name].tolist()
        assert got[:total] == w and got[total:] == [-3] * (tokens - total), name
    assert (d["table"].cpu().numpy() == table).all()
    if index is not None:
        assert (d["kv_index"].cpu().numpy() == index).all()
    assert d["free_left"].tolist() == left and d["free_count"].tolist() == [n_free]


@pytest.mark.parametrize("page", [1, 7, 16, 256])
@pytest.mark.parametrize("lens,news", [([0], [1]), ([5], [0]), ([15, 16, 17, 0], [1, 1, 1, 1]), ([0, 3, 64], [130, 0, 33]),
                                       ([31, 1, 0, 16, 48], [0, 20, 0, 17, 1])])
def test_page_plan(page, lens, news):
    width = -(-max(n + m for n, m in zip(lens, news)) // page) + 1
    check_plan(page, lens, news, width, 200, 200, max(1, sum(news)) + 5)


def test_page_plan_many_requests():
    rng = np.random.default_rng(3)
    lens, news = rng.integers(0, 300, 4096), rng.integers(0, 4, 4096)
    check_plan(16, lens.tolist(), news.tolist(), 20, 3000, 3500, 12288)


@pytest.mark.parametrize("batch", [255, 256, 257, 1024, 1025])
@pytest.mark.parametrize("page", [1, 16])
def test_page_plan_of_as_many_requests_as_threads(batch, page):
    """One request a thread, and several; each token its own row or many rows a request."""
    rng = np.random.default_rng(batch)
    lens, news = rng.integers(0, 40, batch), rng.integers(0, 9, batch)
    news[::3] = 0
    check_plan(page, lens.tolist(), news.tolist(), -(-48 // page), 9 * batch // page, 9 * batch, int(news.sum()) + 3)
    check_plan(page, lens.tolist(), news.tolist(), -(-48 // page), batch // page, 9 * batch, int(news.sum()) - 3)  # too few of both


def test_page_plan_over_several_blocks():
    rng = np.random.default_rng(4)
    lens, news = rng.integers(0, 300, 37), rng.integers(0, 1500, 37)
    check_plan(16, lens.tolist(), news.tolist(), 120, 3000, 3000, 60000, with_index=False)


@pytest.mark.parametrize("n_free", [-2, 0, 3, 50])
def test_page_plan_short_of_pages(n_free):
    """The list runs out inside a request; a count beyond the list is the list's size."""
    check_plan(4, [3, 8, 0, 2], [10, 9, 5, 2], 8, n_free, 5, 40)


def test_page_plan_out_of_room():
    check_plan(4, [3, 30, 100], [40, 9, 5], 4, 20, 20, 60)                   # past the table
    check_plan(4, [3, 30], [40, 9], 16, 20, 20, 60, index_stride=21)         # past the list
    check_plan(4, [3, 8, 1], [10, 9, 5], 8, 20, 20, 12)                      # past the token rows
    check_plan(4, [-3, 2 ** 31 - 3, 5], [4, 9, -2], 8, 20, 20, 40)           # lengths out of range
    check_plan(2, [0, 0, 0], [2 ** 31 - 1, 2 ** 31 - 1, 5], 8, 20, 20, 40)   # sums past 32 bits


def test_page_plan_of_large_page_ids():
    """A cell past 31 bits is no cell."""
    ctx = gpu.DeviceContext(0)
    cells, left = ints([-3] * 3), ints([0, 0])
    gpu.device_page_plan(ctx, 1 << 16, ints([5, 0, 70000]), ints([1, 1, 1]), ints([[32767, 3], [-1, -1], [1, 40000]]),
                         ints([65535]), ints([1]), left, ints([0] * 4), None, None, cells)
    ctx.synchronize()
    assert cells.tolist() == [32767 * 65536 + 5, -1, -1] and left.tolist() == [0, 0]


# ---- the tree plan --------------------------------------------------------------
@pytest.mark.parametrize("kind", ["random", "chain", "roots"])
@pytest.mark.parametrize("counts,max_nodes", [([1], 1), ([8], 8), ([0, 3, 0, 5], 7), ([33, 64, 1], 64), ([65, 100], 100),
                                              ([256, 17], 256)])
def test_tree_plan(kind, counts, max_nodes):
    parents, seen, depth = draft(counts, 5, kind)
    lens = [11 * i for i in range(len(counts))]
    total, spare = len(parents), 4
    words = gpu.tree_words(max_nodes)
    pos, mask = ints([-3] * (total + spare)), ints([[-3] * words] * (total + spare))
    ctx = gpu.DeviceContext(0)
    gpu.device_tree_plan(ctx, starts_of(counts), ints(lens), ints(parents + [0] * spare), max_nodes, pos, mask)
    ctx.synchronize()
    first = np.repeat(lens, counts)
    assert pos.tolist() == [int(n) + d for n, d in zip(first, depth)] + [-3] * spare
    assert (mask.cpu().numpy()[:total] == words_of(seen, words)).all()
    assert (mask.cpu().numpy()[total:] == -3).all()


def test_tree_plan_of_bad_parents():
    """A parent that is no earlier node makes a root; tokens past max_nodes see no node."""
    ctx = gpu.DeviceContext(0)
    pos, mask = ints([-3] * 7), ints([[-3]] * 7)
    gpu.device_tree_plan(ctx, ints([0, 7]), ints([100]), ints([0, 0, 7, 2 ** 31 - 1, -2 ** 31, 3, 2]), 5, pos, mask)
    ctx.synchronize()
    assert mask.flatten().tolist() == [1, 3, 4, 8, 16, 0, 0]
    assert pos.tolist() == [100, 101, 100, 100, 100, 100, 100]


# ---- norm, rotation, store ------------------------------------------------------
def qk_reference(x, gain, dim, neox, steps, pos, factors, eps):
    """(tokens, heads, d) in float64; the angle a float32 product and quotient"""
    y = x.astype(np.float64).copy()
    if gain is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * gain
    theta = pos.astype(np.float32)[:, None] * steps
    if factors is not None:
        theta = theta / factors
    c, s = np.cos(theta.astype(np.float64))[:, None], np.sin(theta.astype(np.float64))[:, None]
    at = np.arange(dim)
    lo, hi = (at[:dim // 2], at[dim // 2:]) if neox else (at[0::2], at[1::2])
    a, b = y[..., lo].copy(), y[..., hi].copy()
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    # rounding: the scale, two products, the angle's cosine and sine, two products and a sum
    size = np.abs(y)
    size[..., lo] = size[..., hi] = np.abs(a) + np.abs(b)
    return y, 8 * 2.0 ** -24 * size + 1e-30


def q8_values(rows, kvw):
    r = rows.cpu()
    q = r[:, :kvw // 2].contiguous().view(torch.int8).numpy().astype(np.float64).reshape(len(r), -1, 32)
    f = r[:, kvw // 2:kvw // 2 + kvw // 32].numpy().astype(np.float64)
    return (q * f[..., None]).reshape(len(r), kvw)


def check_qk(tokens, heads, kv, d, dim, neox, norm, with_factors, form, store=True, in_place=False, live=None, scale=1.0,
             positions=None, pad=3):
    rng = np.random.default_rng(tokens * 7 + d)
    qw, kvw = heads * d, kv * d
    row = (scale * rng.standard_normal((tokens, qw + 2 * kvw + pad))).astype(np.float32)
    steps = gpu.rope_steps(dim, 10000.0)
    gains = [(1 + 0.1 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)] if norm else [None, None]
    factors = np.exp(rng.standard_normal(dim // 2)).astype(np.float32) if with_factors else None
    pos = np.asarray(positions if positions is not None else rng.integers(0, 100000, tokens), np.int32)
    rows = tokens + 6
    cells = rng.permutation(rows)[:tokens].astype(np.int32)
    if tokens > 2:
        cells[1] = -1  # (not stored)
    ctx = gpu.DeviceContext(0)
    dev = torch.from_numpy(row).cuda()
    q, k, v = dev[:, :qw], dev[:, qw:qw + kvw], dev[:, qw + kvw:qw + 2 * kvw]
    q_out = q if in_place else torch.full((tokens, qw + 4), -3.0, device="cuda")[:, :qw]
    k_out = k if in_place else torch.full((tokens, kvw), -3.0, device="cuda")
    crow = gpu.cache_row(FORMS[form], kvw)
    kc, vc = (torch.full((rows, crow), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    more = dict(k_cache=kc, v_cache=vc, cells=ints(cells)) if store else {}
    up = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    gpu.device_qk_norm_rope(ctx, q, k, v if store else None, heads, kv, d, dim, neox, up(steps), ints(pos), q_out, **more,
                            form=FORMS[form], k_out=k_out, q_norm=up(gains[0]), k_norm=up(gains[1]), eps=1e-6,
                            factors=up(factors), count=None if live is None else ints([live]))
    ctx.synchronize()
    n = tokens if live is None else max(0, min(live, tokens))
    for src, got, heads_, gain in ((row[:, :qw], q_out, heads, gains[0]), (row[:, qw:qw + kvw], k_out, kv, gains[1])):
        want, gate = qk_reference(src.reshape(tokens, heads_, d), gain, dim, neox, steps, pos, factors, 1e-6)
        g = got.cpu().numpy().astype(np.float64).reshape(tokens, heads_, d)
        assert (np.abs(g - want) <= gate)[:n].all()
        rest = src.reshape(tokens, heads_, d)[n:] if in_place else -3.0
        assert (g[n:] == rest).all()
    # the cache: halves within half a step of the value, 8-bit rows within half a quant's
    # and their factor's half step
    vals = row[:, qw + kvw:qw + 2 * kvw].astype(np.float64)
    for cache, w in ((kc, want.reshape(tokens, kvw)), (vc, vals)):
        stored = set()
        got = cache.cpu().numpy().astype(np.float64) if form == "f16" else q8_values(cache, kvw)
        for t in range(n):
            if cells[t] < 0 or not store:
                continue
            stored.add(int(cells[t]))
            if form == "f16":
                gate = np.abs(w[t]) * 2.0 ** -11 + 2.0 ** -25 + 8 * 2.0 ** -24 * np.abs(w[t]).max() * 2
            else:
                amax = np.repeat(np.abs(w[t]).reshape(-1, 32).max(1), 32)
                gate = amax * (0.501 / 127 + 2.0 ** -11 + 2.0 ** -20) + 127 * 2.0 ** -25
            assert (np.abs(got[cells[t]] - w[t]) <= gate).all(), t
        others = [i for i in range(rows) if i not in stored]
        assert (cache[others].cpu() == 7.0).all()


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("heads,kv,d,dim", [(4, 2, 64, 64), (8, 1, 128, 128), (2, 2, 32, 32), (4, 1, 96, 48), (3, 3, 128, 90),
                                            (4, 4, 64, 2), (8, 4, 256, 256), (2, 1, 512, 256)])
def test_qk_heads(form, neox, heads, kv, d, dim):
    check_qk(5, heads, kv, d, dim, neox, True, neox, form)


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("heads,kv,d,dim", [(4, 2, 64, 64), (8, 1, 128, 128), (4, 4, 64, 20), (8, 4, 256, 256), (3, 3, 128, 92),
                                            (1, 1, 128, 64), (16, 8, 64, 32), (2, 2, 256, 4)])
def test_qk_aligned_rows(form, neox, heads, kv, d, dim):
    """Rows on 16 bytes (the words of two and four values); head counts that leave a run short."""
    check_qk(5, heads, kv, d, dim, neox, True, neox, form, pad=4)
    check_qk(70, heads, kv, d, dim, neox, False, not neox, form, pad=0)
    check_qk(9, heads, kv, d, dim, neox, True, False, form, pad=4, in_place=True, live=6)


@pytest.mark.parametrize("tokens", [1, 2, 63, 300])
@pytest.mark.parametrize("norm", [False, True])
def test_qk_tokens(tokens, norm):
    check_qk(tokens, 32, 8, 128, 128, True, norm, False, "f16")
    check_qk(tokens, 8, 8, 64, 64, False, norm, True, "q8")


def test_qk_in_place_and_without_caches():
    check_qk(9, 8, 2, 128, 64, True, True, False, "f16", in_place=True)
    check_qk(9, 8, 2, 128, 64, False, True, False, "f16", store=False, in_place=True)
    check_qk(9, 8, 2, 64, 64, False, False, False, "f16", store=False)


@pytest.mark.parametrize("live", [-1, 0, 1, 4, 9, 20])
def test_qk_rows_behind_the_count(live):
    check_qk(9, 8, 2, 128, 128, True, True, False, "f16", live=live)


def test_qk_sizes_of_values_and_positions():
    check_qk(6, 4, 2, 128, 128, True, True, False, "f16", scale=1e4)
    check_qk(6, 4, 2, 64, 64, False, True, False, "q8", scale=1e-3)
    check_qk(4, 4, 2, 64, 64, False, False, False, "f16", positions=[0, 1, 2 ** 24 + 1, 2 ** 31 - 1])


def test_qk_of_zeros():
    """A zero head is zero (eps carries the norm), in either form."""
    ctx = gpu.DeviceContext(0)
    row, out = torch.zeros(2, 4 * 64, device="cuda"), torch.full((2, 128), 3.0, device="cuda")
    gain, steps = torch.ones(64, device="cuda"), torch.from_numpy(gpu.rope_steps(64, 1e4)).cuda()
    for form in FORMS.values():
        kc = torch.ones(2, gpu.cache_row(form, 64), dtype=torch.float16, device="cuda")
        vc = torch.ones_like(kc)
        gpu.device_qk_norm_rope(ctx, row[:, :128], row[:, 128:192], row[:, 192:], 2, 1, 64, 64, True, steps, ints([3, 4]),
                                out, kc, vc, ints([0, 1]), form, q_norm=gain, k_norm=gain)
        ctx.synchronize()
        assert (out == 0).all()
        used = 64 if form == gpu.CACHE_F16 else 34
        assert (kc[:, :used] == 0).all() and (vc[:, :used] == 0).all()


# ---- attention --------------------------------------------------------------------
def encode(x, form):
    if form == "f16":
        return x.half()
    y = x.reshape(x.shape[0], -1, 32)
    amax = y.abs().amax(-1)
    q = torch.trunc(y * (127 / amax)[..., None] + torch.where(y < 0, -0.5, 0.5)).clamp(-127, 127).to(torch.int8)
    kvw = x.shape[1]
    row = torch.zeros(x.shape[0], gpu.cache_row(gpu.CACHE_Q8, kvw), dtype=torch.float16)
    row[:, :kvw // 2] = q.reshape(-1, kvw).view(torch.float16)
    row[:, kvw // 2:kvw // 2 + kvw // 32] = (amax / 127).half()
    return row


class Step:
    """Sequences with their caches and trees on the host, and the attention of a token in float64."""

    def __init__(self, form, lens, counts, heads, kv, d, seed=0, paged=False, kind="random", max_nodes=None, spare=3):
        self.form, self.lens, self.counts, self.heads, self.kv, self.d, self.paged = form, lens, counts, heads, kv, d, paged
        g = torch.Generator().manual_seed(seed)
        self.max_nodes = max_nodes or max(max(counts), 1)
        self.max_count = max(n + m for n, m in zip(lens, counts)) or 1
        self.room = self.max_count + 5
        b = len(lens)
        cells = b * self.room
        self.k, self.v = (encode(torch.randn(cells, kv * d, generator=g), form) for _ in range(2))
        order = torch.randperm(cells, generator=g) if paged else torch.arange(cells)
        self.index = order.reshape(b, self.room).to(torch.int32)
        self.tokens = sum(counts) + spare
        self.q = torch.randn(self.tokens, heads * d, generator=g)
        _, self.seen, _ = draft(counts, seed, kind)
        self.scale = float(np.float32(d ** -0.5))

    def values(self, rows):
        return rows.double() if self.form == "f16" else torch.from_numpy(q8_values(rows, self.kv * self.d))

    def run(self, ctx=None, out=None, work=None):
        ctx = ctx or gpu.DeviceContext(0)
        words = gpu.tree_words(self.max_nodes)
        mask = np.concatenate([words_of(self.seen, words), np.full((self.tokens - len(self.seen), words), -1, np.int32)])
        out = torch.full((self.tokens, self.heads * self.d), -3.0, device="cuda") if out is None else out
        self.dev = dict(q=self.q.cuda(), k=self.k.cuda(), v=self.v.cuda(), starts=starts_of(self.counts),
                        lengths=ints(self.lens), mask=ints(mask), index=self.index.cuda() if self.paged else None)
        e = self.dev
        torch.cuda.synchronize()
        gpu.device_attend_tree(ctx, e["q"], e["k"], e["v"], self.heads, self.kv, self.d, self.scale, e["starts"], e["lengths"],
                               e["mask"], self.max_nodes, self.max_count, out,
                               cache_stride=0 if self.paged else self.room * self.k.shape[1], kv_index=e["index"],
                               form=FORMS[self.form], work=work)
        ctx.synchronize()
        return out.cpu()

    def want(self):
        out = torch.full((self.tokens, self.heads * self.d), -3.0, dtype=torch.float64)
        t = 0
        k, v = self.values(self.k), self.values(self.v)
        for b, (n, m) in enumerate(zip(self.lens, self.counts)):
            for _ in range(m):
                slots = list(range(n)) + [n + i for i in sorted(self.seen[t])]
                rows = [int(self.index[b, j]) for j in slots if int(self.index[b, j]) >= 0]
                for h in range(self.heads):
                    at = slice(h // (self.heads // self.kv) * self.d, (h // (self.heads // self.kv) + 1) * self.d)
                    o = slice(h * self.d, (h + 1) * self.d)
                    if not rows:
                        out[t, o] = 0
                        continue
                    s = k[rows][:, at] @ self.q[t, o].double() * self.scale
                    out[t, o] = torch.softmax(s, 0) @ v[rows][:, at]
                t += 1
        return out

    def check(self, got):
        want = self.want()
        peak = float(self.values(self.v).abs().max())
        assert torch.isfinite(got).all()
        off = (got.double() - want).abs().max()
        assert off <= 1e-5 * peak, float(off)
        assert (got[sum(self.counts):] == -3.0).all()


HEADS = [(2, 2, 64), (4, 2, 128), (8, 2, 64), (8, 1, 128), (4, 4, 32), (8, 2, 96), (4, 2, 256), (2, 1, 512)]


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("heads,kv,d", HEADS)
def test_attend_heads(form, paged, heads, kv, d):
    """Ragged sequences, one with no nodes and one with no context, edges inside a slice."""
    s = Step(form, [70, 0, 33, 5], [9, 7, 0, 1], heads, kv, d, seed=d, paged=paged)
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("length", [0, 1, 31, 32, 63, 64, 65, 127, 128, 1000])
@pytest.mark.parametrize("nodes", [1, 2, 33])
def test_attend_lengths(form, d, length, nodes):
    s = Step(form, [length], [nodes], 4, 1, d, seed=length)
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("heads,kv,d", [(2, 2, 64), (8, 1, 128), (4, 2, 128)])
@pytest.mark.parametrize("counts", [[256], [100, 256], [17, 3, 64, 40, 16, 15]])
def test_attend_large_trees(form, heads, kv, d, counts):
    """Several tiles of rows a sequence; the masks cross words and slices."""
    s = Step(form, [45 + 70 * i for i in range(len(counts))], counts, heads, kv, d, seed=3, paged=len(counts) > 1)
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("nodes", [3, 20])
def test_attend_long(form, heads, kv, d, nodes):
    """Many slices a share."""
    s = Step(form, [20001, 9000], [nodes, nodes - 1], heads, kv, d, seed=8, paged=True)
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 64), (8, 8, 64), (8, 2, 128), (5, 5, 128), (4, 2, 96), (8, 1, 256)])
@pytest.mark.parametrize("length", [500, 2500, 20001])
def test_attend_many_parts(form, heads, kv, d, length):
    """Room for many rows and few of them there: a row in up to 128 parts, folded by
    the kernel for many rows."""
    s = Step(form, [length, 30], [3, 2], heads, kv, d, seed=5, max_nodes=256)
    s.check(s.run())


@pytest.mark.parametrize("kind", ["chain", "roots"])
@pytest.mark.parametrize("form", ["f16", "q8"])
def test_attend_chains_and_roots(kind, form):
    s = Step(form, [40, 100], [50, 64], 4, 2, 64, kind=kind)
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", [(64, 5), (128, 5), (128, 40), (64, 40), (96, 9)])
def test_attend_rows_that_see_nothing(form, d, nodes):
    """No context and an empty mask: zeros; with some seen by others of the same tile."""
    s = Step(form, [0, 6], [nodes, nodes], 4, 2, d)
    for t in (0, 2, nodes - 1):
        s.seen[t] = set()
    s.seen[nodes + 1] = set()  # (sees its context alone)
    got = s.run()
    s.check(got)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", [(64, 6), (128, 6), (128, 45), (64, 45), (256, 6)])
def test_attend_positions_not_held(form, d, nodes):
    s = Step(form, [90, 20], [nodes, 3], 4, 2, d, paged=True)
    s.index[0, 3::5] = -1
    s.index[1, :20] = -1  # (none of its context)
    s.index[1, 21] = -1   # (nor its second node)
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("heads,kv,d,nodes", [(4, 2, 64, 6), (4, 1, 128, 4), (4, 2, 128, 45), (8, 1, 64, 30), (4, 2, 256, 6)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -65504.0])
@pytest.mark.parametrize("paged", [False, True])
def test_attend_ignores_what_is_not_seen(form, heads, kv, d, nodes, bad, paged):
    """What lies in the nodes that a token does not see, in slots behind the
    sequence and in cells that are not held changes no bit of its result."""
    s = Step(form, [70, 30], [nodes, nodes], heads, kv, d, paged=paged)
    for t in range(2 * nodes):  # the last node is seen by itself alone, the one before by nobody
        s.seen[t] -= {nodes - 2}
        if t % nodes != nodes - 1:
            s.seen[t] -= {nodes - 1}
    if paged:
        s.index[0, 11] = -1
        s.index[1, 0] = -1
    clean = s.run()
    s.check(clean)
    kvw = kv * d

    def spoil(cells):
        for c in (s.k, s.v):
            for i in cells:
                if form == "f16":
                    c[i] = bad
                else:
                    c[i, kvw // 2:kvw // 2 + kvw // 32] = bad

    free = [b * s.room + j for b, n in enumerate(s.lens) for j in range(n + nodes, s.room)]
    rows = [int(s.index[b, n + nodes - 2]) for b, n in enumerate(s.lens)] + \
        [int(s.index.reshape(-1)[i]) for i in free]
    if paged:  # cell 0 is what a row that is not held may be read from
        used = set(s.index.reshape(-1).tolist())
        rows += [i for i in range(len(s.k)) if i not in used]
    spoil(rows)
    assert torch.equal(s.run(), clean)
    # seen by one token alone: that one's result goes with it, the others' do not
    spoil([int(s.index[b, n + nodes - 1]) for b, n in enumerate(s.lens)])
    got = s.run()
    last = [nodes - 1, 2 * nodes - 1]
    others = [t for t in range(s.tokens) if t not in last]
    assert torch.equal(got[others], clean[others])
    if bad != bad:
        assert torch.isnan(got[last]).all()
    elif bad == float("inf"):
        assert not torch.isfinite(got[last]).any()


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", [(64, 3), (128, 40), (96, 5)])
def test_attend_scales(form, d, nodes):
    """A negative scale, large queries and queries of very different size."""
    s = Step(form, [50], [nodes], 2, 1, d)
    s.scale = -s.scale
    s.check(s.run())
    s.scale = -s.scale
    s.q[0] *= 1e-6
    s.q[1] = 0
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", [(64, 3), (128, 3), (128, 70), (256, 3), (96, 3)])
@pytest.mark.parametrize("rise", [0.004, 0.08, 1.9, 2.76, 2.85, 5.6, -0.08])
def test_attend_of_rising_scores(form, d, nodes, rise):
    """Scores that rise with the position, by `rise` a key or (from 1 on) a 50th key:
    the running maximum moves at every slice, at some, or by just less and just more
    than what the sums are left alone for."""
    length = 900
    s = Step(form, [length, 40], [nodes, 2], 1, 1, d)
    g = torch.Generator().manual_seed(7)
    along = torch.randn(d, generator=g)
    steps = torch.arange(length, dtype=torch.float32)
    score = rise * (steps if rise < 1 else (steps / 50).floor())
    s.k[:length] = encode((score - score.max() / 2)[:, None] / s.scale * along / (along @ along) +
                          0.02 * torch.randn(length, d, generator=g), form)
    s.q[:nodes] = along * (1 + 0.1 * torch.randn(nodes, 1, generator=g))
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", [(64, 3), (64, 20), (128, 3), (128, 20), (256, 3), (96, 3)])
@pytest.mark.parametrize("length", [0, 20, 40, 64, 100, 130])
@pytest.mark.parametrize("size", [1e4, 1e-3])
def test_attend_of_large_and_small_values(form, d, nodes, length, size):
    """Values far from 1, with a context that ends anywhere in a slice."""
    s = Step(form, [length, 70], [nodes, 2], 4, 2, d, seed=length, paged=True)
    g = torch.Generator().manual_seed(2)
    s.v = encode(size * torch.randn(len(s.v), 2 * d, generator=g).clamp(-6, 6), form)
    s.k = encode(2 * torch.randn(len(s.k), 2 * d, generator=g), form)
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", [(64, 3), (64, 30), (128, 3), (128, 30), (128, 70), (256, 3), (96, 3)])
@pytest.mark.parametrize("first,last", [(1e-4, 3e3), (3e3, 1e-4)])
def test_attend_of_values_whose_size_moves(form, d, nodes, first, last):
    """Values that grow or shrink along the positions, in each 32 of them at a place of
    its own; a few queries look at the small ones alone, held to those."""
    length = 700
    s = Step(form, [length, 33], [nodes, 3], 2, 1, d, seed=11)
    g = torch.Generator().manual_seed(12)
    cells, blocks = len(s.v), d // 32
    place = (torch.arange(cells)[:, None] + 40 * torch.arange(blocks)[None, :]).clamp(max=length) / length
    size = first * (last / first) ** place
    s.v = encode((torch.randn(cells, blocks, 32, generator=g) * size[..., None]).reshape(cells, d), form)
    s.check(s.run())
    small = slice(0, 60) if first < last else slice(640, length)
    s.k[:length] = encode(0.01 * torch.randn(length, d, generator=g), form)
    along = torch.randn(d, generator=g)
    s.k[small] = encode(along * (50 / s.scale) / (along @ along) + 0.01 * torch.randn(60, d, generator=g), form)
    s.q[0] = along.repeat(2)
    got, want = s.run(), s.want()
    s.check(got)
    # the others' weights are 2^-72 of these
    assert (got[0].double() - want[0]).abs().max() <= 1e-5 * float(s.values(s.v)[small].abs().max())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", [(64, 3), (128, 40), (96, 5), (256, 2)])
def test_attend_without_a_scale(form, d, nodes):
    """Every key weighs the same."""
    s = Step(form, [50, 0], [nodes, 1], 2, 1, d)
    s.scale = 0.0
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", [(64, 4), (128, 4), (128, 70), (256, 4), (96, 4)])
def test_attend_scores_past_an_exponent(form, d, nodes):
    """One query whose scores are near 1e8, where a weight's exponent has no
    fraction left: the key it points at takes all of it, the other queries are as
    without it."""
    s = Step(form, [700], [nodes], 1, 1, d)
    s.k[333] = encode(torch.full((1, d), 4.0), form)[0]
    plain = s.run()
    s.check(plain)
    s.q[2] = 1e7
    got = s.run()
    others = [t for t in range(nodes) if t != 2]
    assert torch.equal(got[others], plain[others])
    assert (got[2].double() - s.values(s.v)[333]).abs().max() <= 1e-5 * float(s.values(s.v).abs().max())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("d,nodes", [(64, 5), (128, 5), (128, 70), (256, 5), (96, 5)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attend_of_a_query_that_is_not_finite(form, d, nodes, bad):
    s = Step(form, [90], [nodes], 2, 1, d)
    clean = s.run()
    s.q[1, d + 3] = bad  # (token 1, head 1)
    got = s.run()
    assert torch.isnan(got[1, d:]).all() and torch.equal(got[1, :d], clean[1, :d])
    others = [t for t in range(s.tokens) if t != 1]
    assert torch.equal(got[others], clean[others])


@pytest.mark.parametrize("form,heads,kv,d", [("f16", 2, 1, 64), ("q8", 2, 1, 128), ("f16", 4, 2, 128), ("f16", 2, 2, 96), ("q8", 1, 1, 256)])
@pytest.mark.parametrize("batch", [64, 65, 200])
def test_attend_many_sequences(form, heads, kv, d, batch):
    """More sequences than a wave has lanes; some without nodes, some without a context."""
    rng = np.random.default_rng(batch)
    lens, counts = rng.integers(0, 70, batch), rng.integers(0, 4, batch)
    lens[::7], counts[3::5], counts[-1] = 0, 0, 2
    s = Step(form, lens.tolist(), counts.tolist(), heads, kv, d, paged=True)
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("only", [0, 63, 64, 150, 299])
def test_attend_one_of_many(form, only):
    counts = [0] * 300
    counts[only] = 7
    s = Step(form, [20] * only + [900] + [20] * (299 - only), counts, 2, 1, 64)
    s.check(s.run())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("d", [128, 96])
def test_cache_past_32_bits(form, paged, d):
    """Cache rows whose offsets pass 2^31 halves and 2^32 bytes, stored and attended."""
    ctx = gpu.DeviceContext(0)
    row = gpu.cache_row(FORMS[form], d)
    cells = (1 << 31) // row + 2000
    pool = [torch.empty(cells, row, dtype=torch.float16, device="cuda") for _ in range(2)]
    s = Step(form, [70, 40], [5, 6], 2, 1, d, paged=True)
    base = [cells - s.room, 5] if paged else [0, cells - s.room]
    for b in range(2):
        at = s.index[b].long()
        pool[0][base[b]:base[b] + s.room] = s.k[at].cuda()
        pool[1][base[b]:base[b] + s.room] = s.v[at].cuda()
    index = torch.stack([torch.arange(s.room) + base[b] for b in range(2)]).to(torch.int32).cuda()
    # the last node's key and value of both sequences by the store
    tokens = torch.randn(2, 4 * d, generator=torch.Generator().manual_seed(3)).cuda()
    last = [n + m - 1 for n, m in zip(s.lens, s.counts)]
    to = ints([int(index[b, last[b]]) for b in range(2)])
    steps = torch.from_numpy(gpu.rope_steps(d, 10000.0)).cuda()
    gpu.device_qk_norm_rope(ctx, tokens[:, :2 * d], tokens[:, 2 * d:3 * d], tokens[:, 3 * d:], 2, 1, d, d, False, steps, ints([0, 0]),
                            torch.empty(2, 2 * d, device="cuda"), pool[0], pool[1], to, FORMS[form])
    ctx.synchronize()
    for b in range(2):
        cell = int(s.index[b, last[b]])
        for c, have, part in ((s.k, pool[0], tokens[b, 2 * d:3 * d]), (s.v, pool[1], tokens[b, 3 * d:])):
            c[cell] = encode(part.cpu()[None], form)[0]
            used = d if form == "f16" else d // 2 + d // 32
            assert torch.equal(have[int(to[b])][:used].cpu().view(torch.int16), c[cell][:used].view(torch.int16))
    words = gpu.tree_words(s.max_nodes)
    mask = ints(np.concatenate([words_of(s.seen, words), np.full((s.tokens - len(s.seen), words), -1, np.int32)]))
    out = torch.full((s.tokens, 2 * d), -3.0, device="cuda")
    gpu.device_attend_tree(ctx, s.q.cuda(), pool[0], pool[1], 2, 1, d, s.scale, starts_of(s.counts), ints(s.lens), mask, s.max_nodes,
                           s.max_count, out, cache_stride=0 if paged else base[1] * row, kv_index=index if paged else None,
                           form=FORMS[form])
    ctx.synchronize()
    s.check(out.cpu())


def test_attend_workspace_contents():
    """A workspace of NaN changes nothing, nor does a larger one."""
    for lens, counts, heads, kv, d in (([300, 0], [5, 0], 8, 2, 128), ([4000, 10], [40, 2], 8, 2, 64), ([90, 4], [3, 9], 4, 2, 96)):
        s = Step("f16", lens, counts, heads, kv, d)
        want = s.run()
        need = 64 << 20
        work = torch.full((need // 4,), float("nan"), device="cuda").view(torch.uint8)
        assert torch.equal(s.run(work=work), want)
        s.check(want)


def test_attend_strided_queries():
    ctx = gpu.DeviceContext(0)
    s = Step("f16", [40, 3], [5, 6], 4, 2, 128)
    want = s.run(ctx)
    row = torch.zeros(s.tokens, 4 * 128 + 2 * 256, device="cuda")
    row[:, :512] = s.q.cuda()
    out = torch.full_like(s.q, -3.0).cuda()
    e = s.dev
    gpu.device_attend_tree(ctx, row[:, :512], e["k"], e["v"], 4, 2, 128, s.scale, e["starts"], e["lengths"], e["mask"],
                           s.max_nodes, s.max_count, out, cache_stride=s.room * s.k.shape[1])
    ctx.synchronize()
    assert torch.equal(out.cpu(), want)


def test_attend_holds_device_values_to_the_checked_sizes():
    """More nodes, longer lengths or later starts than the host was told: no row
    past the buffers, and what is left of the sequence is attended."""
    ctx = gpu.DeviceContext(0)
    s = Step("f16", [40, 30], [5, 4], 4, 2, 64, spare=0)
    s.run(ctx)
    e = s.dev
    guard = torch.full((s.tokens + 8, 256), -3.0, device="cuda")
    out = guard[:s.tokens]
    for starts, lengths in (([0, 5, 200], [40, 30]), ([0, 5, 9], [4000, -7]), ([-4, 12, 3], [40, 30])):
        gpu.device_attend_tree(ctx, e["q"], e["k"], e["v"], 4, 2, 64, s.scale, ints(starts), ints(lengths), e["mask"],
                               s.max_nodes, s.max_count, out, cache_stride=s.room * s.k.shape[1])
        ctx.synchronize()
        assert (guard[s.tokens:] == -3.0).all() and torch.isfinite(guard).all()


# ---- a run of them ------------------------------------------------------------------
class Draft:
    """Two layers' worth of a step: plan, norm + rotation + store, attention, on paged caches."""

    def __init__(self, ctx, form, heads=8, kv=2, d=64, page=16):
        self.ctx, self.form, self.heads, self.kv, self.d, self.page = ctx, form, heads, kv, d, page
        self.lens, self.counts = [37, 0, 64], [7, 5, 0]
        self.parents, self.seen, self.depth = draft(self.counts, 4)
        g = torch.Generator().manual_seed(1)
        self.tokens, self.max_nodes, self.max_count = 16, 8, 72
        self.row = torch.randn(self.tokens, (heads + 2 * kv) * d, generator=g).cuda()
        self.gain = [(1 + 0.1 * torch.randn(d, generator=g)).cuda() for _ in range(2)]
        self.steps = torch.from_numpy(gpu.rope_steps(d, 10000.0)).cuda()
        pages = torch.randperm(24, generator=g).to(torch.int32)
        width = -(-self.max_count // page)
        self.table = torch.full((3, width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(self.lens):
            h = -(-n // page)
            self.table[b, :h] = pages[at:at + h]
            at += h
        self.free = pages[at:].cuda()
        j = torch.arange(width * page)
        cell = self.table[:, j // page] * page + (j % page).int()
        self.index = torch.where(j < torch.tensor(self.lens)[:, None], cell, -1).to(torch.int32).cuda()
        self.table = self.table.cuda()
        self.k, self.v = (encode(torch.randn(24 * page, kv * d, generator=g), form).cuda() for _ in range(2))
        self.i = dict(lengths=ints(self.lens), news=ints(self.counts), n_free=ints([self.free.numel()]), left=ints([0, 0]),
                      starts=ints([0] * 4), cells=ints([-3] * self.tokens), slots=ints([-3] * self.tokens),
                      parents=ints(self.parents + [0] * (self.tokens - len(self.parents))), pos=ints([0] * self.tokens),
                      mask=ints([[0]] * self.tokens))
        self.q = torch.zeros(self.tokens, heads * d, device="cuda")
        self.out = torch.full((self.tokens, heads * d), -3.0, device="cuda")

    def step(self):
        i, qw, kvw = self.i, self.heads * self.d, self.kv * self.d
        gpu.device_page_plan(self.ctx, self.page, i["lengths"], i["news"], self.table, self.free, i["n_free"], i["left"],
                             i["starts"], None, i["slots"], i["cells"], self.index)
        gpu.device_tree_plan(self.ctx, i["starts"], i["lengths"], i["parents"], self.max_nodes, i["pos"], i["mask"])
        gpu.device_qk_norm_rope(self.ctx, self.row[:, :qw], self.row[:, qw:qw + kvw], self.row[:, qw + kvw:], self.heads,
                                self.kv, self.d, self.d, True, self.steps, i["pos"], self.q, self.k, self.v, i["cells"],
                                FORMS[self.form], q_norm=self.gain[0], k_norm=self.gain[1], count=i["starts"][3:])
        gpu.device_attend_tree(self.ctx, self.q, self.k, self.v, self.heads, self.kv, self.d, 0.125, i["starts"],
                               i["lengths"], i["mask"], self.max_nodes, self.max_count, self.out, kv_index=self.index,
                               form=FORMS[self.form])

    def check(self):
        total, d = sum(self.counts), self.d
        qw = self.heads * d
        pos = np.repeat(self.lens, self.counts) + np.array(self.depth)
        row = self.row.cpu().numpy()[:total]
        q, _ = qk_reference(row[:, :qw].reshape(total, self.heads, d), self.gain[0].cpu().numpy(), d, True, self.steps.cpu().numpy(),
                            pos, None, 1e-5)
        val = lambda c: c.cpu().double() if self.form == "f16" else torch.from_numpy(q8_values(c, self.kv * d))  # noqa: E731
        k, v, index = val(self.k), val(self.v), self.index.cpu()
        t = 0
        for b, (n, m) in enumerate(zip(self.lens, self.counts)):
            for _ in range(m):
                rows = index[b, list(range(n)) + [n + i for i in sorted(self.seen[t])]].tolist()
                assert min(rows) >= 0
                for h in range(self.heads):
                    at = slice(h // (self.heads // self.kv) * d, (h // (self.heads // self.kv) + 1) * d)
                    s = k[rows][:, at] @ torch.from_numpy(q[t, h]) * 0.125
                    w = torch.softmax(s, 0) @ v[rows][:, at]
                    assert (self.out[t, h * d:(h + 1) * d].cpu().double() - w).abs().max() <= 1e-5 * float(v.abs().max())
                t += 1
        assert (self.out[total:] == -3.0).all()
        return self.out.clone()


@pytest.mark.parametrize("form", ["f16", "q8"])
def test_step(form):
    ctx = gpu.DeviceContext(0)
    s = Draft(ctx, form)
    s.step()
    ctx.synchronize()
    s.check()


def test_step_on_another_stream():
    stream = torch.cuda.Stream()
    ctx = gpu.DeviceContext(0, stream)
    s = Draft(ctx, "f16")
    torch.cuda.synchronize()
    s.step()
    ctx.synchronize()
    s.check()


def test_step_captured_and_replayed():
    """One graph serves every size of the step: other lengths, trees and pages
    between the replays, eager work in between, each replay against the eager step;
    a second context's graph beside it."""
    sets = []
    for form in ("f16", "q8"):
        stream = torch.cuda.Stream()
        ctx = gpu.DeviceContext(0, stream)
        s = Draft(ctx, form)
        torch.cuda.synchronize()
        s.step()
        ctx.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            s.step()
        sets.append((s, g, ctx))
    for lens, counts in (([37, 0, 64], [7, 5, 0]), ([37, 0, 64], [1, 0, 8]), ([20, 0, 64], [8, 8, 0]), ([37, 0, 60], [0, 0, 0])):
        for s, g, ctx in sets:
            s.lens, s.counts = lens, counts
            s.parents, s.seen, s.depth = draft(counts, 9)
            s.i["lengths"].copy_(ints(lens))
            s.i["news"].copy_(ints(counts))
            s.i["parents"][:len(s.parents)].copy_(ints(s.parents))
            s.out.fill_(-3.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(ctx.stream):
                g.replay()
            ctx.synchronize()
            got = s.check()
            s.out.fill_(-3.0)
            torch.cuda.synchronize()
            s.step()
            ctx.synchronize()
            assert torch.equal(s.out, got)


def test_a_workspace_that_grows_leaves_a_captured_one():
    """A graph replays on the workspace it was captured with, also after larger
    calls on the same context have replaced it."""
    stream = torch.cuda.Stream()
    ctx = gpu.DeviceContext(0, stream)
    s = Draft(ctx, "f16")
    torch.cuda.synchronize()
    s.step()
    ctx.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        s.step()
    held = ctx._work
    ctx.workspace(held.numel() * 4)
    assert ctx._work is not held and any(w is held for w in ctx._captured)
    with torch.cuda.stream(stream):
        g.replay()
    ctx.synchronize()
    s.check()


def test_python_refusals():
    ctx = gpu.DeviceContext(0)
    s = Step("f16", [4], [2], 2, 1, 64)
    s.run(ctx)
    e = s.dev
    out = torch.zeros(s.tokens, 128, device="cuda")

    def attend(**k):
        a = dict(q=e["q"], k_cache=e["k"], v_cache=e["v"], heads=2, kv_heads=1, head_dim=64, scale=0.1, starts=e["starts"],
                 lengths=e["lengths"], mask=e["mask"], max_nodes=2, max_count=6, out=out)
        gpu.device_attend_tree(ctx, **{**a, **k})

    attend()
    for bad in (dict(q=e["q"].cpu()), dict(q=e["q"].half()), dict(q=e["q"].t()), dict(k_cache=e["k"][:3].contiguous()),
                dict(v_cache=e["v"].float()), dict(starts=e["starts"].long()), dict(starts=e["starts"][:1]),
                dict(mask=e["mask"][:1].contiguous()), dict(out=out[:2]), dict(out=out.t()), dict(max_nodes=300),
                dict(kv_index=ints([1, 2, 3])), dict(out=e["q"]),
                dict(work=torch.empty(1 << 24, dtype=torch.uint8)), dict(work=torch.empty(1 << 22, device="cuda"))):
        with pytest.raises((ValueError, gpu.MiError)):
            attend(**bad)
    with pytest.raises(ValueError):
        gpu.device_tree_plan(ctx, e["starts"], e["lengths"], ints([0] * 5), 2, None, ints([0] * 4))
    with pytest.raises(ValueError):
        gpu.device_page_plan(ctx, 16, ints([1, 2]), ints([1]), ints([[1], [2]]), ints([1]), ints([1]), ints([0, 0]),
                             ints([0] * 3), None, None, ints([0]))
    n = ints([1, 0])
    for left, page in ((n, 16), (ints([0, 0]), 0)):  # free_left in free_count's place; pages of nothing
        with pytest.raises(gpu.MiError):
            gpu.device_page_plan(ctx, page, ints([1]), ints([1]), ints([[1]]), ints([1]), n[:1], left, ints([0, 0]), None,
                                 None, ints([0]))
