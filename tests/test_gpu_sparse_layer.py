"""The decoder layer with sparse experts and a window (mi_layer_desc experts,
window) against a float64 layer, token by token, under the per-element layer gate
of tests/layer64.py: decode batches, a sequence's chunk, both cache forms and
layouts, trees, chained layers and a captured step."""

import numpy as np
import pytest
import torch

import oracle
from molla_amd import block, gpu, synth
from molla_amd._lib import MiError
from tests import layer64 as l64
from tests import npquant
from tests.test_gpu_tree import FORMS, encode, q8_values

pytestmark = pytest.mark.gpu

SHAPE = dict(width=256, heads=4, kv_heads=2, head_dim=64, rope_dim=64, rope_base=10000.0, eps=1e-5)


class Layer:
    """One layer on the device, and the same weights in float64."""

    def __init__(self, kinds=(gpu.Q_Q4_K, gpu.Q_Q4_K, gpu.Q_Q6_K), hidden=512, experts=6, used=2, flags=gpu.ROUTER_NORM,
                 bias=False, window=0, first=0, post=False, qk_norm=False, act=0, seed=1, **shape):
        s = dict(SHAPE, **shape)
        self.spec = block.BlockSpec(**s, hidden=hidden, experts=experts, experts_used=used, router_flags=flags,
                                    router_scale=1.25, window=window, first=first, act=act)
        w, qw, kvw = s["width"], s["heads"] * s["head_dim"], s["kv_heads"] * s["head_dim"]
        shapes = dict(wq=(kinds[0], qw, w), wk=(kinds[0], kvw, w), wv=(kinds[0], kvw, w), wo=(kinds[0], w, qw))
        if experts:
            shapes.update(gate=(kinds[1], experts * hidden, w), up=(kinds[1], experts * hidden, w),
                          down=(kinds[2], experts * w, hidden))
        else:
            shapes.update(gate=(kinds[1], hidden, w), up=(kinds[1], hidden, w), down=(kinds[2], w, hidden))
        self.W, weights = {}, {}
        for i, (n, (kind, r, c)) in enumerate(shapes.items()):
            blob = synth.quant_tensor(kind, r, c, seed * 100 + i)
            weights[n] = gpu.Tensor.from_bytes(blob, kind, c, r)
            self.W[n] = npquant.dequant(kind, blob.numpy(), r * c).reshape(r, c).astype(np.float64)
        v = lambda n, k, mean=0.0, std=1.0: synth.normal(n, seed * 100 + k, mean=mean, std=std)
        self.vec = dict(attn_norm=v(w, 50, 1.0, 0.1), ffn_norm=v(w, 51, 1.0, 0.1))
        extras = {}
        if experts:
            extras["router"] = v(experts * w, 52, std=0.3)
            if bias:
                extras["router_bias"] = v(experts, 53, std=0.1)
        if post:
            extras.update(attn_post_norm=v(w, 54, 1.0, 0.1), ffn_post_norm=v(w, 55, 1.0, 0.1))
        if qk_norm:
            extras.update(q_norm=v(s["head_dim"], 56, 1.0, 0.1), k_norm=v(s["head_dim"], 57, 1.0, 0.1))
        self.vec.update(extras)
        self.layer = block.DeviceLayer(self.spec, self.vec["attn_norm"].cuda(), self.vec["ffn_norm"].cuda(), weights,
                                       torch.from_numpy(gpu.rope_steps(s["rope_dim"], s["rope_base"])).cuda(),
                                       extras={k: t.cuda() for k, t in extras.items()})

    def token64(self, x, pos, rows):
        """A token's output and its gate; rows(k, v): the cache rows it sees, given its own."""
        s, W = self.spec, self.W
        f = {k: t.double().numpy() for k, t in self.vec.items()}
        n = l64.rms64(x, f["attn_norm"], s.eps)
        q, k, v = W["wq"] @ n, W["wk"] @ n, W["wv"] @ n
        if "q_norm" in f:
            q = np.concatenate([l64.rms64(h, f["q_norm"], s.eps) for h in q.reshape(s.heads, -1)])
            k = np.concatenate([l64.rms64(h, f["k_norm"], s.eps) for h in k.reshape(s.kv_heads, -1)])
        q = l64.rope64(q, s.heads, s.head_dim, s.rope_dim, s.rope_base, False, pos, None)
        k = l64.rope64(k, s.kv_heads, s.head_dim, s.rope_dim, s.rope_base, False, pos, None)
        keys, values = rows(k, v)
        attn = l64.attend64(q, keys.reshape(-1), values.reshape(-1), len(keys), s.heads, s.kv_heads, s.head_dim, s.attn_scale)
        y, post = W["wo"] @ attn, {}
        if "attn_post_norm" in f:
            post["attn"] = (y, f["attn_post_norm"])
            y = l64.rms64(y, f["attn_post_norm"], s.eps)
        x = x + y
        n = l64.rms64(x, f["ffn_norm"], s.eps)
        fn = l64.gelu64 if s.act else l64.silu64
        if not s.experts:
            act = fn(W["gate"] @ n) * (W["up"] @ n)
            down = W["down"]
        else:
            logits = f["router"].reshape(s.experts, -1) @ n
            if s.router_flags & gpu.ROUTER_SIGMOID:
                p = 1 / (1 + np.exp(-logits))
            else:
                p = np.exp(logits - logits.max())
                p /= p.sum()
            score = p + f.get("router_bias", 0.0)
            order = np.argsort(-score, kind="stable")
            ids = order[:s.experts_used]
            # (the choice is a step: a test whose choice hangs on rounding shows nothing.  A
            # normed row that is off by 2^-19 of itself moves a logit by that of sum |r n|,
            # about 256 * 0.24 * 0.8 = 49: 1e-4, and a quarter of it through a sigmoid)
            if s.experts_used < s.experts:
                last, next_ = order[s.experts_used - 1], order[s.experts_used]
                if s.router_flags & gpu.ROUTER_SIGMOID:
                    assert score[last] - score[next_] > 2.5e-5
                else:
                    assert logits[last] - logits[next_] > 1e-4
            g = p[ids] * s.router_scale
            if s.router_flags & gpu.ROUTER_NORM:
                g = g / p[ids].sum()
            H = s.hidden
            # the weighted experts end to end: one long row of each
            down = np.concatenate([W["down"][e * s.width:(e + 1) * s.width] * g[i] for i, e in enumerate(ids)], 1)
            act = np.concatenate([fn(W["gate"][e * H:(e + 1) * H] @ n) * (W["up"][e * H:(e + 1) * H] @ n) for e in ids])
        y = down @ act
        if "ffn_post_norm" in f:
            post["ffn"] = (y, f["ffn_post_norm"])
            y = l64.rms64(y, f["ffn_post_norm"], s.eps)
        parts = dict(W=dict(wo=W["wo"], down=down), attn=attn, act=act, post=post, eps=s.eps)
        return x + y, l64.layer_bound(parts)


class Run:
    def __init__(self, layer, lens, form, paged, chunk=0, seed=4):
        """Sequences of `lens` positions and a token more each; or one of lens[0] and a chunk of `chunk`."""
        self.l, self.form, self.paged, self.chunk = layer, form, paged, chunk
        s = layer.spec
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.kvw = len(lens), s.kv_width()
        self.room = max(lens) + (chunk or 1) + 3
        self.k, self.v = (encode(torch.randn(self.seqs * self.room, self.kvw, generator=g), form).cuda() for _ in range(2))
        self.pos = [lens[0] + i for i in range(chunk)] if chunk else list(lens)
        self.index = torch.randperm(self.seqs * self.room, generator=g).int().view(self.seqs, self.room) if paged else None
        self.x = torch.randn(len(self.pos), s.width, generator=g)

    def go(self, ctx):
        n, s = len(self.pos), self.l.spec
        x, pos = self.x.cuda().clone(), torch.tensor(self.pos, dtype=torch.int32, device="cuda")
        if self.paged:
            block.device_layer_paged(ctx, self.l.layer, x, self.k, self.v, self.index.cuda(), 0 if self.chunk else self.room,
                                     pos, self.room, n, form=FORMS[self.form])
        else:
            block.device_layer(ctx, self.l.layer, x, self.k, self.v, 0 if self.chunk else self.room * self.k.shape[1], pos,
                               self.room, n, form=FORMS[self.form])
        torch.cuda.synchronize()
        return x

    def check(self, x, rows=None):
        s, got = self.l.spec, x.cpu().numpy()
        k, v = ((t.cpu().double().numpy() if self.form == "f16" else q8_values(t, self.kvw)) for t in (self.k, self.v))
        for t in rows or range(len(self.pos)):
            b, p = (0 if self.chunk else t), self.pos[t]
            j = np.arange(p + 1)
            if s.window:
                j = j[(j > p - s.window) | (j < s.first)]
            at = self.index[b].numpy()[j] if self.paged else b * self.room + j
            want, bound = self.l.token64(self.x[t].double().numpy(), p, lambda key, val: (k[at], v[at]))
            err = np.abs(got[t] - want)
            assert (err <= bound).all(), (t, (err / bound).max())


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("lens", [(70,), (90, 3, 41), (60, 0, 33, 10, 21, 99, 7, 50)])
@pytest.mark.parametrize("window,first", [(0, 0), (16, 2)])
def test_decode(form, paged, lens, window, first):
    r = Run(Layer(window=window, first=first), lens, form, paged)
    r.check(r.go(gpu.DeviceContext(0)))


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("chunk,start", [(5, 20), (12, 0), (77, 30)])
@pytest.mark.parametrize("window,first", [(0, 0), (24, 3)])
def test_chunk(form, paged, chunk, start, window, first):
    r = Run(Layer(window=window, first=first), (start,), form, paged, chunk)
    r.check(r.go(gpu.DeviceContext(0)), rows=sorted({0, 1, chunk // 2, chunk - 1}))


@pytest.mark.parametrize("kw", [
    dict(experts=0, window=16, first=1), dict(kinds=(gpu.Q_Q8_0,) * 3, window=8),
    dict(kinds=(gpu.Q_Q4_K, gpu.Q_Q5_K, gpu.Q_Q4_0), flags=gpu.ROUTER_SIGMOID | gpu.ROUTER_NORM, bias=True),
    dict(flags=gpu.ROUTER_SIGMOID, used=6), dict(post=True, qk_norm=True, window=9, first=4), dict(act=gpu.ACT_BIT, used=1),
    dict(hidden=256, experts=40, used=8), dict(head_dim=256, rope_dim=256, heads=2, kv_heads=1, window=20),
    dict(head_dim=96, rope_dim=96, heads=8, kv_heads=2, window=20, first=2, width=768)])
@pytest.mark.parametrize("tokens", ["one", "four", "chunk"])
def test_families(kw, tokens):
    lens, chunk = {"one": ((44,), 0), "four": ((44, 5, 19, 30), 0), "chunk": ((40,), 20)}[tokens]
    r = Run(Layer(**kw), lens, "f16", False, chunk)
    r.check(r.go(gpu.DeviceContext(0)))


def test_workspace_is_what_the_layer_takes():
    """A layer on exactly its workspace, among bytes that stay as they were."""
    for lens, chunk in (((70,), 0), ((90, 3, 41), 0), ((30,), 50)):
        r = Run(Layer(window=16, first=2), lens, "f16", False, chunk)
        n = len(r.pos)
        need = block.layer_workspace(r.l.layer, r.room, n)
        held = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
        x, pos = r.x.cuda().clone(), torch.tensor(r.pos, dtype=torch.int32, device="cuda")
        stride = 0 if chunk else r.room * r.k.shape[1]
        block.device_layer(gpu.DeviceContext(0), r.l.layer, x, r.k, r.v, stride, pos, r.room, n, work=held[256:256 + need])
        torch.cuda.synchronize()
        assert (held[:256] == 77).all() and (held[256 + need:] == 77).all()
        r.check(x)
        with pytest.raises(MiError):
            block.device_layer(gpu.DeviceContext(0), r.l.layer, x, r.k, r.v, stride, pos, r.room, n,
                               work=held[256:256 + need - 256])


def test_chained_layers_and_a_captured_step():
    """A session of sparse windowed layers: prefill, decode, and the captured step's picks."""
    layers = [Layer(window=16, first=2, seed=s) for s in (1, 2, 3)]
    spec = layers[0].spec
    vocab = 512
    head = gpu.Tensor.from_bytes(synth.quant_tensor(gpu.Q_Q6_K, vocab, spec.width, 9), gpu.Q_Q6_K, spec.width, vocab)
    model = block.DeviceModel(spec, synth.normal(vocab * spec.width, 5, "cuda").view(vocab, spec.width),
                              [l.layer for l in layers], synth.normal(spec.width, 6, "cuda", mean=1.0, std=0.1), head)
    picks = []
    for captured in (False, True):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            ses = block.DeviceSession(gpu.DeviceContext(0, stream), model, 3, 128)
            for b in range(3):
                ses.prefill(synth.tokens(40 + 7 * b, vocab, 30 + b).cuda(), b)
            ses.finish()
            ses.advance()
            ses.step(advance=True)
            out = [ses.picks.clone()]
            graph = ses.capture() if captured else None
            for _ in range(12):
                graph.replay() if captured else ses.step(advance=True)
                out.append(ses.picks.clone())
            ses.ctx.synchronize()
        picks.append(torch.stack(out))
    assert torch.equal(picks[0], picks[1])
    assert len(set(picks[0].flatten().tolist())) > 3


def test_experts_over_trees_of_drafts():
    """A tree of one path is a chunk: the same layer over both."""
    l = Layer()
    n, m = 21, 6
    ctx = gpu.DeviceContext(0)
    r = Run(l, (n,), "f16", False, m)
    k0, v0 = r.k.clone(), r.v.clone()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    starts, lengths, parents = i32([0, m]), i32([n]), i32(list(range(-1, m - 1)))
    pos, mask = i32([0] * m), torch.zeros(m, 1, dtype=torch.int32, device="cuda")
    gpu.device_tree_plan(ctx, starts, lengths, parents, m, pos, mask)
    x = r.x.cuda().clone()
    block.device_layer_tree(ctx, l.layer, x, k0, v0, starts, lengths, mask, pos, i32([n + i for i in range(m)]), m, r.room)
    torch.cuda.synchronize()
    r.k, r.v = k0, v0
    r.check(x)
    w = Layer(window=8)
    with pytest.raises(MiError, match="window"):
        block.device_layer_tree(ctx, w.layer, x, k0, v0, starts, lengths, mask, pos, i32([n + i for i in range(m)]), m, r.room,
                                work=torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
