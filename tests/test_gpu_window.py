"""Attention over a window and the first positions (mi_attend_window) against
float64 over the values the caches hold.

The bound: a score is off by its 3 * head_dim / 16 sums (and about 16 more of a
q8_0 cache's factors) of 2^-24 of the absolute products, which moves a weight, and
so the result, by twice that of the largest value; the weighted sum by 2^-24 of the
largest value for each of its 2 products a 16 keys, and about 64 rescalings and
roundings.
"""

import math

import pytest
import torch

from molla_amd import gpu, synth
from tests.test_gpu_tree import FORMS, encode, q8_values

pytestmark = pytest.mark.gpu


def values(rows, form, kvw):
    return rows.double() if form == "f16" else torch.from_numpy(q8_values(rows.cpu(), kvw)).to(rows.device)


class Case:
    def __init__(self, seqs, room, heads, kv_heads, head_dim, form, paged, seed=1, qpad=0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kvh, self.d, self.form = heads, kv_heads, head_dim, form
        self.kvw, self.room = kv_heads * head_dim, room
        self.k, self.v = (encode(torch.randn(seqs * room, self.kvw, generator=g), form).cuda() for _ in range(2))
        self.index = torch.randperm(seqs * room, generator=g).int().view(seqs, room).cuda() if paged else None
        self.g, self.qpad = g, qpad
        self.scale = 1.0 / math.sqrt(head_dim)

    def run(self, pos, window, first, chunk, max_count=None, ctx=None, q=None):
        t, qw = len(pos), self.heads * self.d
        if q is None:
            q = torch.randn(t, qw + self.qpad, generator=self.g).cuda()[:, :qw]
        self.q = q
        out = torch.full((t, qw), 9.0, device="cuda")
        index = self.index
        if index is not None and chunk:
            index = index[0]
        gpu.device_attend_window(ctx or gpu.DeviceContext(0), q, self.k, self.v, self.heads, self.kvh, self.d, self.scale,
                                 window, first, torch.tensor(pos, dtype=torch.int32, device="cuda"), max_count or self.room,
                                 out, cache_stride=0 if chunk else self.room * self.k.shape[1], kv_index=index,
                                 form=FORMS[self.form])
        return out

    def seen(self, row, p, window, first, chunk):
        """Cache rows that the token at p of sequence `row` sees."""
        b = 0 if chunk else row
        j = torch.arange(max(p + 1, 0), device="cuda")
        j = j[(j > p - window) | (j < first)]
        if self.index is None:
            return j + b * self.room
        cells = self.index[b, j].long()
        return cells[cells >= 0]

    def check(self, out, pos, window, first, chunk, rows=None):
        k, v = values(self.k, self.form, self.kvw), values(self.v, self.form, self.kvw)
        for t in rows if rows is not None else range(len(pos)):
            at = self.seen(t, pos[t], window, first, chunk)
            if not at.numel():
                assert (out[t] == 0).all()
                continue
            kk, vv = (x[at].view(-1, self.kvh, self.d).transpose(0, 1).contiguous() for x in (k, v))
            q = self.q[t].double().view(self.kvh, -1, self.d)
            s = torch.matmul(q, kk.transpose(1, 2).contiguous()) * self.scale
            want = torch.matmul(torch.softmax(s, -1), vv).reshape(-1)
            big = vv.abs().max().item()
            size = (torch.matmul(q.abs(), kk.abs().transpose(1, 2).contiguous()) * self.scale).max().item()
            bound = 2.0 ** -24 * big * (2 * (3 * self.d / 16 + 16) * size + at.numel() / 8 + 64)
            err = (out[t].double() - want).abs().max().item()
            assert err <= bound, (t, err, bound)


SHAPES = [(8, 2, 128), (8, 8, 64), (8, 1, 64), (4, 2, 256), (8, 2, 96), (2, 1, 32)]


@pytest.mark.parametrize("heads,kvh,d", SHAPES)
@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("window,first", [(1, 0), (7, 1), (64, 4), (100, 70), (33, 300), (5000, 4)])
def test_decode(heads, kvh, d, form, paged, window, first):
    c = Case(7, 500, heads, kvh, d, form, paged, qpad=8)
    pos = [0, 1, 63, 64, 99, 320, 499]
    c.check(c.run(pos, window, first, False), pos, window, first, False)


@pytest.mark.parametrize("heads,kvh,d", SHAPES)
@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("window,first", [(1, 0), (7, 1), (64, 4), (150, 70), (33, 300), (5000, 0)])
@pytest.mark.parametrize("start,n", [(0, 40), (300, 133)])
def test_chunk(heads, kvh, d, form, paged, window, first, start, n):
    c = Case(1, 450, heads, kvh, d, form, paged, qpad=4)
    pos = list(range(start, start + n))
    c.check(c.run(pos, window, first, True), pos, window, first, True, rows=list(range(0, n, 11)) + [n - 1])


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("window,first", [(1000, 4), (4096, 0), (64, 1000), (2**31 - 1, 2**31 - 1)])
def test_long_contexts(form, chunk, window, first):
    """Several shares and splits, two slices' ends inside the window."""
    n = 9 if chunk else 3
    c = Case(1 if chunk else n, 9000, 8, 2, 128, form, chunk)
    pos = [8990 + i for i in range(n)] if chunk else [8999, 4101, 1003]
    c.check(c.run(pos, window, first, chunk), pos, window, first, chunk)


@pytest.mark.parametrize("d,kvh", [(128, 2), (64, 4), (256, 1), (96, 2)])
@pytest.mark.parametrize("form", ["f16", "q8"])
def test_small_chunks_and_many_sequences(d, kvh, form):
    c = Case(1, 400, 8, kvh, d, form, False)
    pos = [100, 101, 102]  # a chunk of few tokens
    c.check(c.run(pos, 50, 2, True), pos, 50, 2, True)
    c = Case(20, 150, 8, kvh, d, form, True)
    pos = [(37 * i) % 150 for i in range(20)]  # more sequences than a decode batch
    c.check(c.run(pos, 50, 2, False), pos, 50, 2, False)


@pytest.mark.parametrize("d", [128, 256, 96])
@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("chunk", [False, True])
def test_rows_that_see_nothing(d, form, chunk):
    n = 12
    c = Case(1 if chunk else n, 200, 4, 2, d, form, True)
    pos = [150 + i for i in range(n)]
    c.index[:, 100:] = -1  # the window's positions are not held
    c.check(c.run(pos, 40, 0, chunk), pos, 40, 0, chunk)
    c.check(c.run(pos, 40, 3, chunk), pos, 40, 3, chunk)
    c.index[0, 1] = -1  # a first one neither
    c.check(c.run(pos, 55, 3, chunk), pos, 55, 3, chunk)
    pos[3], pos[7] = -1, -2**31  # padding
    c.check(c.run(pos, 55, 3, chunk), pos, 55, 3, chunk)
    out = c.run([-1] * n, 55, 3, chunk)
    assert (out == 0).all()


def test_positions_past_the_context_are_its_last():
    for n, chunk in ((3, False), (12, True)):
        c = Case(1 if chunk else n, 64, 4, 2, 64, "f16", False)
        out = c.run([70, 2**31 - 1] + [63] * (n - 2), 20, 1, chunk, max_count=64)
        c.check(out, [63] * n, 20, 1, chunk)


@pytest.mark.parametrize("d", [128, 256, 96])
@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("chunk,paged", [(False, True), (True, True), (True, False)])
def test_what_is_not_seen_changes_nothing(d, form, chunk, paged):
    n, room = 12, 400
    c = Case(1 if chunk else n, room, 4, 2, d, form, paged)
    pos = [300 + i for i in range(n)]
    if paged:
        c.index[:, 290] = -1
    q = torch.randn(n, 4 * d, generator=c.g).cuda()
    base = c.run(pos, 100, 4, chunk, q=q)
    c.check(base, pos, 100, 4, chunk)
    unseen = torch.ones(c.k.shape[0], dtype=torch.bool, device="cuda")
    for t in range(n):
        unseen[c.seen(t, pos[t], 100, 4, chunk)] = False
    assert unseen.any()
    for bits in (0x7c00, -0x0400, 0x7e01):  # infinities, NaN; of a q8_0 row its factors too
        for x in (c.k, c.v):
            x.view(torch.int16)[unseen] = bits
        assert torch.equal(c.run(pos, 100, 4, chunk, q=q), base)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 40])
def test_values_that_are_not_finite(d, n):
    """They reach the rows that see them, at their place, and no other."""
    c = Case(1, 300, 4, 2, d, "f16", n == 40)
    pos = list(range(200, 200 + n))
    q = torch.randn(n, 4 * d, generator=c.g).cuda()
    window, first = 30, 2
    base = c.run(pos, window, first, True, q=q).view(n, 2, 2, d)
    hit = {180: (0, 3, float("inf")), 199: (1, d - 1, float("-inf")), 1: (1, 17, float("nan")), 215: (0, 40, float("inf"))}
    for j, (kvh, at, bad) in hit.items():
        c.v[c.index[0, j].long() if c.index is not None else j, kvh * d + at] = bad
    out = c.run(pos, window, first, True, q=q).view(n, 2, 2, d)
    touched = torch.zeros(n, 2, 2, d, dtype=torch.bool, device="cuda")
    for t, p in enumerate(pos):
        for j, (kvh, at, _) in hit.items():
            if j <= p and (j > p - window or j < first):
                touched[t, kvh, :, at] = True
    assert not torch.isfinite(out[touched]).any()
    # (a row that sees one may take another path to its other places)
    big = c.v[torch.isfinite(c.v)].abs().max().item()
    assert torch.isfinite(out[~touched]).all()
    assert (out - base)[~touched].abs().max().item() <= 2.0 ** -18 * big
    clean = ~touched.flatten(1).any(1)
    assert torch.equal(out[clean], base[clean])


@pytest.mark.parametrize("chunk", [False, True])
def test_cells_past_32_bits(chunk):
    """A pool of more than 2^31 halves."""
    cells, kvh, d, n = (1 << 21) + 700, 8, 128, 10
    c = Case(1, 8, 8, kvh, d, "f16", False)
    c.k, c.v = (torch.zeros(cells, kvh * d, dtype=torch.float16, device="cuda") for _ in range(2))
    at = torch.cat([torch.arange(300), torch.arange(cells - 300, cells)])[torch.randperm(600, generator=c.g)].int().cuda()
    for x in (c.k, c.v):
        x[at.long()] = torch.randn(600, kvh * d, generator=c.g).half().cuda()
    c.room = 600
    c.index = at[None].repeat(1 if chunk else n, 1).contiguous()
    pos = [560 + i for i in range(n)]
    out = c.run(pos, 200, 5, chunk)
    hold, index = (c.k, c.v), c.index
    c.k, c.v = (x[at.long()] for x in hold)  # the same rows, without the gap
    c.index = torch.arange(600, device="cuda", dtype=torch.int32)[None].repeat(index.shape[0], 1)
    c.check(out, pos, 200, 5, chunk)


def test_most_tokens():
    c = Case(1, 128, 1, 1, 64, "f16", False)
    pos = [i % 128 for i in range(65536)]
    out = c.run(pos, 9, 2, True)
    c.check(out, pos, 9, 2, True, rows=[0, 1, 127, 128, 40000, 65535])
    c = Case(1, 128, 1, 1, 64, "f16", True)
    c.index = c.index.repeat(65536, 1)
    out = c.run(pos, 9, 2, False)
    c.index = c.index[:1]
    c.check(out, pos, 9, 2, True, rows=[0, 1, 127, 128, 40000, 65535])


def test_large_scores():
    """A rising run of scores of thousands: the running maximum moves in every slice."""
    for n, chunk in ((4, False), (64, True)):
        c = Case(1 if chunk else n, 900, 8, 2, 128, "f16", False)
        ramp = (torch.arange(c.k.shape[0]) % 900).float() / 30
        c.k[:, ::128] = ramp[:, None].half().cuda()
        q = torch.randn(n, 8 * 128, generator=c.g).cuda()
        q[:, ::128] = 300.0
        pos = [800 + i for i in range(n)]
        c.check(c.run(pos, 500, 10, chunk, q=q), pos, 500, 10, chunk, rows=range(0, n, 3))


def test_captured_and_on_another_stream():
    s = torch.cuda.Stream()
    ctx = gpu.DeviceContext(0, s)
    for n, chunk in ((3, False), (40, True)):
        c = Case(1 if chunk else n, 300, 8, 2, 128, "f16", True)
        q = torch.randn(n, 8 * 128, generator=c.g).cuda()
        pos = torch.zeros(n, dtype=torch.int32, device="cuda")
        out, eager = torch.zeros(n, 1024, device="cuda"), torch.zeros(n, 1024, device="cuda")
        index = c.index[0] if chunk else c.index
        torch.cuda.synchronize()

        def step(o):
            gpu.device_attend_window(ctx, q, c.k, c.v, 8, 2, 128, c.scale, 77, 3, pos, 300, o, kv_index=index)

        with torch.cuda.stream(s):
            step(out)
            ctx.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step(out)
        for at in (0, 90, 255):
            with torch.cuda.stream(s):
                pos.copy_(at + torch.arange(n, device="cuda", dtype=torch.int32))
                out.zero_()
                g.replay()
                step(eager)
            ctx.synchronize()
            assert torch.equal(out, eager)
            c.q = q
            c.check(out, [at + i for i in range(n)], 77, 3, chunk, rows=[0, n - 1])
