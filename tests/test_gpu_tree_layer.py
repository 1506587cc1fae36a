"""The decoder layer over trees of drafted tokens on the GPU
(mi_decoder_layer_tree): against a float64 layer in which every token attends
over the cache rows its path has, under the per-element layer gate of
tests/layer64.py; the rows it stores; padded batches; a captured step of plans and
layers."""

import numpy as np
import pytest
import torch

import oracle
from molla_amd import block, gpu
from tests import layer64 as l64
from tests.test_gpu_families import FAMILIES, device_family_layer, family_host, oracle_spec
from tests.test_gpu_layer import assert_layer_close, device_layer_from, make_layer_weights, spec_of
from tests.test_gpu_tree import FORMS, draft, encode, ints, q8_values

pytestmark = pytest.mark.gpu


def token64(spec, host, W, x, pos, rows):
    """One token through the layer in float64.  rows(k, v): the key and value rows
    its path has, its own among them, given its own.  Returns the output and the
    parts of l64.layer_bound."""
    H, KV, HD, eps = spec["heads"], spec["kv_heads"], spec["head_dim"], spec["eps"]
    f = {k: np.asarray(host[k], np.float64) for k in oracle.OPTIONAL_VECTORS + ("attn_norm", "ffn_norm") if host.get(k) is not None}
    x = x.astype(np.float64)
    n = l64.rms64(x, f["attn_norm"], eps)
    q, k, v = W["wq"] @ n, W["wk"] @ n, W["wv"] @ n
    if "q_bias" in f:
        q, k, v = q + f["q_bias"], k + f["k_bias"], v + f["v_bias"]
    if "q_norm" in f:
        q = np.concatenate([l64.rms64(h, f["q_norm"], eps) for h in q.reshape(H, HD)])
        k = np.concatenate([l64.rms64(h, f["k_norm"], eps) for h in k.reshape(KV, HD)])
    fac = host.get("rope_factors")
    q = l64.rope64(q, H, HD, spec["rope_dim"], spec["rope_base"], spec["neox"], pos, fac)
    k = l64.rope64(k, KV, HD, spec["rope_dim"], spec["rope_base"], spec["neox"], pos, fac)
    keys, values = rows(k, v)
    attn = l64.attend64(q, keys.reshape(-1), values.reshape(-1), len(keys), H, KV, HD, spec["attn_scale"])
    post = {}
    y = W["wo"] @ attn
    if "attn_post_norm" in f:
        post["attn"] = (y, f["attn_post_norm"])
        y = l64.rms64(y, f["attn_post_norm"], eps)
    x = x + y
    n = l64.rms64(x, f["ffn_norm"], eps)
    fn = l64.gelu64 if spec.get("act") else l64.silu64
    u = W["up"] @ n
    act = fn(u) if spec.get("ungated") else fn(W["gate"] @ n) * u
    y = W["down"] @ act
    if "ffn_post_norm" in f:
        post["ffn"] = (y, f["ffn_post_norm"])
        y = l64.rms64(y, f["ffn_post_norm"], eps)
    return x + y, {"W": W, "attn": attn, "act": act, "post": post, "eps": eps}


class Trees:
    """A step's trees over caches of either layout, planned on the device."""

    def __init__(self, ctx, spec, lens, counts, form, paged, seed=3, spare=0, max_nodes=None, layers=1):
        self.ctx, self.lens, self.counts, self.form, self.paged = ctx, lens, counts, form, paged
        self.kvw = spec["kv_heads"] * spec["head_dim"]
        g = torch.Generator().manual_seed(seed)
        b = len(lens)
        self.max_nodes = max_nodes or max(counts)
        self.max_count = max(n + m for n, m in zip(lens, counts))
        self.page = 16 if paged else self.max_count + 4  # one page a sequence: its own cache
        self.width = -(-(self.max_count + 4) // self.page)  # pages of a sequence
        self.room = self.width * self.page
        self.tokens = sum(counts) + spare
        self.parents, self.seen, self.depth = draft(counts, seed)
        pages = torch.randperm(b * self.width, generator=g) if paged else torch.arange(b * self.width)
        table = pages.reshape(b, self.width).to(torch.int32)
        held = torch.arange(self.width) < -(-torch.tensor(lens) // self.page)[:, None]
        self.free = table[~held].flip(0).contiguous().cuda()
        self.table = torch.where(held, table, -1).to(torch.int32).cuda()
        at = (table[:, :, None] * self.page + torch.arange(self.page)).reshape(b, self.room)
        self.index = torch.where(torch.arange(self.room) < torch.tensor(lens)[:, None], at, -1).to(torch.int32).cuda()
        self.k, self.v = ([encode(torch.randn(b * self.room, self.kvw, generator=g), form).cuda() for _ in range(layers)]
                          for _ in range(2))
        self.x = torch.randn(self.tokens, spec["width"], generator=g)
        self.i = dict(lengths=ints(lens), news=ints(counts), starts=ints([0] * (b + 1)), cells=ints([-3] * self.tokens),
                      parents=ints(self.parents + [0] * spare), pos=ints([1 << 20] * self.tokens),
                      mask=ints([[-1] * gpu.tree_words(self.max_nodes)] * self.tokens), many=ints([self.free.numel()]), left=ints([0, 0]))
        self.xd = self.x.cuda()

    def plan(self):
        i = self.i
        gpu.device_page_plan(self.ctx, self.page, i["lengths"], i["news"], self.table, self.free, i["many"], i["left"],
                             i["starts"], None, None, i["cells"], self.index)
        gpu.device_tree_plan(self.ctx, i["starts"], i["lengths"], i["parents"], self.max_nodes, i["pos"], i["mask"])

    def layer(self, layer, at=0, work=None):
        i = self.i
        block.device_layer_tree(self.ctx, layer, self.xd, self.k[at], self.v[at], i["starts"], i["lengths"], i["mask"], i["pos"],
                                i["cells"], self.max_nodes, self.max_count,
                                cache_stride=0 if self.paged else self.room * self.k[at].shape[1],
                                kv_index=self.index if self.paged else None, form=FORMS[self.form], work=work)

    def values(self, rows):
        return rows.cpu().double().numpy() if self.form == "f16" else q8_values(rows, self.kvw)

    def check(self, spec, host, before):
        """xd and the caches after one layer against float64; before: the caches' values then"""
        got = self.xd.cpu().numpy()
        k, v, index = self.values(self.k[0]), self.values(self.v[0]), self.index.cpu().numpy()
        W = {n: l64.dq(host[n]) for n in ("wq", "wk", "wv", "wo", "gate", "up", "down") if n in host}
        new = np.zeros(len(k), bool)
        t = 0
        for b, (n, m) in enumerate(zip(self.lens, self.counts)):
            for i in range(m):
                cell = index[b, n + i]
                new[cell] = True

                def rows(key, value):
                    for have, want in ((k[cell], key), (v[cell], value)):
                        # f16: half a step of the value; q8_0: half a step of its 32
                        # values' largest over 127, whose factor is an f16 of its own;
                        # beside them 1e-4 of the row's scale for the f32 products
                        big = np.abs(want).reshape(-1, 32).max(1).repeat(32)
                        step = np.abs(want) * 2.0 ** -11 if self.form == "f16" else big * (0.5 / 127 + 2.0 ** -11)
                        assert (np.abs(have - want) <= step + 1e-3 * np.sqrt(np.mean(want * want))).all()
                    at = index[b, list(range(n)) + [n + j for j in sorted(self.seen[t])]]
                    return k[at], v[at]

                out, parts = token64(spec, host, W, self.x[t].numpy(), n + self.depth[t], rows)
                assert_layer_close(got[t], out, l64.layer_bound(parts), f"sequence {b} node {i}:")
                t += 1
        for have, was in zip((k, v), before):
            assert np.array_equal(have[~new], was[~new])  # no other row is written


def run(spec, host, layer, lens, counts, form, paged, **kw):
    ctx = gpu.DeviceContext(0)
    s = Trees(ctx, spec, lens, counts, form, paged, **kw)
    before = [s.values(c[0]).copy() for c in (s.k, s.v)]
    s.plan()
    s.layer(layer)
    ctx.synchronize()
    s.check(spec, host, before)
    return s


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("lens,counts", [([33], [1]), ([20], [6]), ([15, 0, 40], [3, 4, 1]), ([20, 0, 40], [13, 5, 0]),
                                         ([31, 16], [40, 20])])
def test_llama_layer(form, paged, lens, counts):
    spec = spec_of(512, 1024, 8, 2, 64)
    host = make_layer_weights(spec, 21)
    _, layer = device_layer_from(host, spec)
    run(spec, host, layer, lens, counts, form, paged)


@pytest.mark.parametrize("name", list(FAMILIES))
@pytest.mark.parametrize("counts", [[3, 4], [9, 12]])
def test_family_layer(name, counts):
    spec, host = family_host(name, spec_of(512, 1024, 8, 2, 64, base=1000000.0), 31)
    spec = oracle_spec(spec)
    _, layer = device_family_layer(spec, host)
    run(spec, host, layer, [18, 7], counts, "f16", True)


@pytest.mark.parametrize("counts", [[2, 3], [9, 8]])
def test_neox_layer_with_wide_heads(counts):
    spec, host = family_host("qwen3", dict(spec_of(512, 1024, 4, 2, 128), neox=1), 33)
    spec = oracle_spec(spec)
    _, layer = device_family_layer(spec, host)
    run(spec, host, layer, [25, 3], counts, "q8", True)


@pytest.mark.parametrize("counts,spare", [([2, 3], 2), ([7, 9], 5)])
def test_rows_behind_the_last_sequence(counts, spare):
    """They hold NaN; no other row and no cache row changes for that."""
    spec = spec_of(512, 1024, 8, 2, 64)
    host = make_layer_weights(spec, 22)
    _, layer = device_layer_from(host, spec)
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        ctx = gpu.DeviceContext(0)
        s = Trees(ctx, spec, [12, 30], counts, "f16", True, spare=spare)
        s.xd[sum(counts):] = fill
        need = 1 << 24
        work = torch.full((need,), 255 if fill != 0 else 0, dtype=torch.uint8, device="cuda")
        s.plan()
        s.layer(layer, work=work)
        ctx.synchronize()
        outs.append((s.xd[:sum(counts)].clone(), s.k[0], s.v[0]))
    for other in outs[1:]:
        for a, b in zip(outs[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("counts", [[3, 2], [4, 4], [9, 2]])
def test_chained_layers(counts):
    """Layers that norm for the next one give the same bits."""
    spec = spec_of(512, 1024, 8, 2, 64)
    outs = []
    for chained in (False, True):
        ctx = gpu.DeviceContext(0)
        layers = [device_layer_from(make_layer_weights(spec, 50 + i), spec)[1] for i in range(3)]
        if chained:
            block.chain_layers([layer.desc for layer in layers])
        s = Trees(ctx, spec, [12, 30], counts, "f16", True, layers=3)
        s.plan()
        for i, layer in enumerate(layers):
            s.layer(layer, i)
        ctx.synchronize()
        outs.append([s.xd] + s.k + s.v)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    """Two contexts' layers in turn on streams of their own, each as it is alone."""
    spec = spec_of(512, 1024, 8, 2, 64)
    _, layer = device_layer_from(make_layer_weights(spec, 60), spec)
    want = []
    for seed in (3, 4):
        ctx = gpu.DeviceContext(0)
        s = Trees(ctx, spec, [200, 900], [20, 13], "f16", True, seed=seed)
        s.plan()
        s.layer(layer)
        ctx.synchronize()
        want.append(s.xd.clone())
    sets = [Trees(gpu.DeviceContext(0, torch.cuda.Stream()), spec, [200, 900], [20, 13], "f16", True, seed=seed) for seed in (3, 4)]
    torch.cuda.synchronize()
    for s in sets:
        s.plan()
    for s in sets:
        s.layer(layer)
    for s, w in zip(sets, want):
        s.ctx.synchronize()
        assert torch.equal(s.xd, w)


@pytest.mark.parametrize("counts", [[3, 2], [8, 6]])
def test_step_captured_and_replayed(counts):
    """Plans and two layers as one graph: other lengths and trees between the
    replays, each against the eager step."""
    spec = spec_of(512, 1024, 8, 2, 64)
    stream = torch.cuda.Stream()
    ctx = gpu.DeviceContext(0, stream)
    layers = [device_layer_from(make_layer_weights(spec, 40 + i), spec)[1] for i in range(2)]
    s = Trees(ctx, spec, [20, 33], counts, "f16", True, layers=2)
    state = s.k + s.v + [s.table, s.index]
    was = [t.clone() for t in state]

    def step():
        s.plan()
        for i, layer in enumerate(layers):
            s.layer(layer, i)

    def reset():
        torch.cuda.synchronize()
        s.xd.copy_(s.x)
        for t, w in zip(state, was):
            t.copy_(w)
        torch.cuda.synchronize()

    torch.cuda.synchronize()
    step()
    ctx.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        step()
    for seed, (lens, now) in enumerate((([20, 33], counts), ([9, 0], counts), ([20, 30], [counts[0], 0]), ([1, 33], [1, counts[1]]))):
        parents, _, _ = draft(now, seed)
        s.i["lengths"].copy_(ints(lens))
        s.i["news"].copy_(ints(now))
        s.i["parents"][:len(parents)].copy_(ints(parents))
        outs = []
        for how in ("replay", "eager"):
            reset()
            if how == "replay":
                with torch.cuda.stream(stream):
                    g.replay()
            else:
                step()
            ctx.synchronize()
            outs.append([s.xd[:sum(now)].clone()] + [t.clone() for t in s.k + s.v])
        for a, b in zip(*outs):
            assert torch.equal(a, b)


def test_python_refusals():
    spec = spec_of(256, 512, 4, 2, 64)
    _, layer = device_layer_from(make_layer_weights(spec, 5), spec)
    ctx = gpu.DeviceContext(0)
    s = Trees(ctx, spec, [4], [3], "f16", True)
    s.plan()
    i = s.i
    good = dict(x=s.xd, k_cache=s.k[0], v_cache=s.v[0], starts=i["starts"], lengths=i["lengths"], mask=i["mask"], pos=i["pos"],
                cells=i["cells"], max_nodes=s.max_nodes, max_count=s.max_count, kv_index=s.index)
    block.device_layer_tree(ctx, layer, **good)
    ctx.synchronize()
    for bad in (dict(x=s.xd[:2]), dict(x=s.xd.double()), dict(cells=i["cells"][:2]), dict(mask=i["mask"][:1]),
                dict(kv_index=s.index[0]), dict(kv_index=None, max_count=1000), dict(starts=i["starts"][:1]), dict(max_nodes=0),
                dict(pos=i["pos"].long()), dict(k_cache=s.k[0].float()), dict(work=torch.empty(64, dtype=torch.uint8, device="cuda")),
                dict(work=torch.empty(1 << 26, dtype=torch.uint8))):
        with pytest.raises((ValueError, gpu.MiError)):
            block.device_layer_tree(ctx, layer, **{**good, **bad})
