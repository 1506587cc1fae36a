"""The decoder layer of sparse-expert families over long contexts, operator by operator.

  router   which experts a token takes, and with which weights
           (gpu.device_router): logits, scores, the largest few
  product  matrix products grouped by expert over quantized weights
           (gpu.device_experts_matmul): a row of x against the matrix that its id names
  mlp      the experts' gated MLP and the weighted sum of what they give
           (gpu.device_experts_mlp)
  window   attention over the last `window` positions and the first few
           (gpu.device_attend_window): one token for each of some sequences, or
           one sequence's chunk, over both cache forms, contiguous and paged

`own` false: the same in elementary torch operations.  Which experts a token
takes is skewed, as trained routers leave it, so that the experts' shares are
ragged; weights are GGUF blocks as a model file holds them.
"""

from __future__ import annotations

import math

import torch

own = False

F16, Q8 = "f16", "q8"
Q4_0, Q8_0, Q4_K, Q6_K = 2, 8, 12, 14  # ggml type numbers
BLOCK = {Q4_0: (32, 18), Q8_0: (32, 34), Q4_K: (256, 144), Q6_K: (256, 210)}  # (values, bytes)


def listed():
    return [
        # a decoding token of a model with many small experts: the latency of the call
        dict(name="router 1 token", op="router", tokens=1, width=2048, experts=64, used=8, sigmoid=False, bias=False,
             norm=True),
        # a long prompt chunk, scores by sigmoid with a balancing bias
        dict(name="router 2048 tokens", op="router", tokens=2048, width=4096, experts=128, used=8, sigmoid=True,
             bias=True, norm=True),
        # one projection of a batch of eight sequences, two large experts each
        dict(name="product 16 rows 8 x 14336x4096", op="product", kind=Q4_K, experts=8, rows=14336, cols=4096, pairs=16,
             share=2),
        # a prompt's rows over many small experts, the second projection (a row of its own each), odd count
        dict(name="product 2403 rows 64 x 2048x1024", op="product", kind=Q6_K, experts=64, rows=2048, cols=1024,
             pairs=2403, share=1),
        # a decoding token, two of eight large experts, the kinds of a Q4_K_M file
        dict(name="mlp 1 token 2 of 8", op="mlp", tokens=1, experts=8, used=2, width=4096, hidden=14336, kind=Q4_K,
             down=Q6_K),
        # a decoding token, eight of 64 small experts
        dict(name="mlp 1 token 8 of 64", op="mlp", tokens=1, experts=64, used=8, width=2048, hidden=1024, kind=Q4_K,
             down=Q4_K),
        # eight sequences decoding together, 8-bit weights
        dict(name="mlp 8 tokens 8 of 64", op="mlp", tokens=8, experts=64, used=8, width=2048, hidden=1024, kind=Q8_0,
             down=Q8_0),
        # a prompt chunk of odd length over large experts
        dict(name="mlp 509 tokens 2 of 8", op="mlp", tokens=509, experts=8, used=2, width=4096, hidden=14336, kind=Q4_K,
             down=Q6_K),
        # one sequence decoding far into a long context
        dict(name="window 1 token at 32768", op="window", tokens=1, chunk=False, heads=32, kv_heads=8, head_dim=128,
             length=32768, window=4096, first=4, form=F16, paged=False),
        # eight sequences of unequal lengths, 8-bit paged cache, odd sizes
        dict(name="window 8 tokens at 9001 q8", op="window", tokens=8, chunk=False, heads=32, kv_heads=8, head_dim=128,
             length=9001, window=1023, first=4, form=Q8, paged=True),
        # a prompt chunk behind a long context
        dict(name="window 256 chunk at 16384", op="window", tokens=256, chunk=True, heads=32, kv_heads=8, head_dim=128,
             length=16384, window=4096, first=4, form=F16, paged=False),
        # a long chunk of a small model (heads of 64, eight query heads a key head), paged
        dict(name="window 2048 chunk at 8192 d64", op="window", tokens=2048, chunk=True, heads=32, kv_heads=4,
             head_dim=64, length=8192, window=1024, first=64, form=F16, paged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["router", "product", "mlp", "mlp", "window", "window"])
    if op == "router":
        experts = rng.choice([8, 16, 60, 64, 128, 256])
        return dict(op="router", tokens=_log(rng, 1, 2048), width=256 * rng.randint(2, 16), experts=experts,
                    used=rng.randint(1, min(experts, 12)), sigmoid=rng.random() < 0.4, bias=rng.random() < 0.4,
                    norm=rng.random() < 0.7)
    if op == "window":
        kv = rng.choice([1, 2, 4, 8])
        chunk = rng.random() < 0.5
        case = dict(op="window", tokens=_log(rng, 9, 2048) if chunk else _log(rng, 1, 16), chunk=chunk,
                    heads=kv * rng.choice([1, 2, 4, 8]), kv_heads=kv, head_dim=rng.choice([64, 64, 128, 128, 128, 256]),
                    length=_log(rng, 16, 32768), window=_log(rng, 1, 8192), first=rng.choice([0, 1, 4, 64, _log(rng, 1, 500)]),
                    form=rng.choice([F16, F16, Q8]), paged=rng.random() < 0.5)
        if chunk:
            case["length"] = max(case["length"], case["tokens"])
            while work(case)["flops"] > 3.6e10 or case["heads"] * case["tokens"] * case["length"] > 7e8:
                case["tokens"] = case["tokens"] * 3 // 4
        return case
    kind = rng.choice([Q4_0, Q8_0, Q4_K, Q4_K, Q6_K])
    experts = rng.choice([4, 8, 16, 60, 64, 128])
    # weights, rows and tokens that keep the products below the listed ones'
    if op == "product":
        rows, cols = 128 * _log(rng, 2, 112), 256 * _log(rng, 2, 56)
        while experts * rows * cols > 4.7e8:
            rows = max(256, rows // 256 * 128)
            cols = max(512, cols // 512 * 256)
        used = rng.randint(1, 8)
        tokens = min(_log(rng, 1, 2048), int(4e10 / (2 * rows * cols * used)) + 1)
        case = dict(op="product", kind=kind, experts=experts, rows=rows, cols=cols, pairs=tokens * used,
                    share=rng.choice([1, used]))
        while work(case)["bytes"] > 9e8:
            case["experts"] -= case["experts"] // 4
        return case
    width, hidden = 256 * _log(rng, 2, 16), 256 * _log(rng, 2, 56)
    while experts * width * hidden > 4.7e8:
        hidden = max(512, hidden // 512 * 256)
        experts = experts if hidden > 512 else experts // 2
    used = rng.randint(1, min(8, experts))
    tokens = min(_log(rng, 1, 1024), int(3e11 / (6 * width * hidden * used)) + 1)
    case = dict(op="mlp", tokens=tokens, experts=experts, used=used, width=width, hidden=hidden, kind=kind,
                down=rng.choice([kind, Q6_K]))
    while work(case)["bytes"] > 9e8:
        case["experts"] -= case["experts"] // 4
        case["used"] = min(case["used"], case["experts"])
    return case


# ---- inputs ----------------------------------------------------------------
class _Inputs:
    """Draws from one seed, in the order asked."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, mean=0.0, std=1.0):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=torch.float32) * std + mean

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def matrix(self, kind, rows, cols):
        """rows x cols weights of a standard deviation of about 1 / sqrt(cols), as (rows, bytes a row)."""
        per, size = BLOCK[kind]
        n = rows * cols // per
        # (bytes by whole words)
        b = torch.randint(-2**31, 2**31, ((n * size + 3) // 4,), generator=self.g, device="cuda", dtype=torch.int64)
        b = b.to(torch.int32).view(torch.uint8)[:n * size].reshape(n, size)

        def factor(std):  # of a block: halves of one sign, a spread of a few times
            f = torch.exp(0.3 * self.normal(n)) * (std / math.sqrt(cols))
            return f.half().view(torch.int16).view(torch.uint8).reshape(n, 2)

        if kind == Q8_0:
            b[:, 0:2] = factor(1 / 74.0)
        elif kind == Q4_0:
            b[:, 0:2] = factor(1 / 4.6)
        elif kind == Q4_K:  # (its minimum takes out the mean of its scaled codes)
            b[:, 0:2] = factor(1 / 190.0)
            b[:, 2:4] = factor(7.5 / 190.0)
            b[:, 8:12] = b[:, 4:8]
            b[:, 12:16] = (b[:, 12:16] & 15) * 17
        else:
            b[:, 192:208] = self.ints(-64, 64, n, 16).to(torch.int8).view(torch.uint8)
            b[:, 208:210] = factor(1 / 680.0)
        return b.reshape(rows, -1)

    def choice(self, tokens, experts, used):
        """Which experts each token takes: some more popular than others."""
        liked = self.normal(experts, std=0.7)
        noise = torch.rand(tokens, experts, generator=self.g, device="cuda").clamp(min=1e-12)
        return (liked - torch.log(-torch.log(noise))).topk(used, 1).indices.to(torch.int32).contiguous()

    def cache(self, form, cells, kv_width):
        """`cells` positions of a cache of either form: (cells, halves a position)."""
        v = self.normal(cells, kv_width)
        if form == F16:
            return v.half()
        x = v.reshape(-1, kv_width // 32, 32)
        amax = x.abs().amax(-1)
        row = torch.zeros(cells, _row(form, kv_width), dtype=torch.float16, device="cuda")
        q = torch.round(x * (127.0 / amax)[..., None]).to(torch.int8)
        row[:, :kv_width // 2] = q.reshape(cells, kv_width).view(torch.float16)
        row[:, kv_width // 2:kv_width // 2 + kv_width // 32] = (amax / 127.0).half()
        return row


def _row(form, kv_width):
    """Halves a cached position takes: halves, or bytes, then a half for each 32, rounded up to 8."""
    return kv_width if form == F16 else (kv_width // 2 + kv_width // 32 + 7) // 8 * 8


def _ends(case):
    """The position of each token: a chunk's last ones, or one of each sequence, unequal."""
    n, t = case["length"], case["tokens"]
    return [n - t + i for i in range(t)] if case["chunk"] else [n - 1 - i * (n // (2 * t)) for i in range(t)]


def _inputs(case, g):
    op = case["op"]
    if op == "router":
        t, w, e = case["tokens"], case["width"], case["experts"]
        return dict(x=g.normal(t, w), router=g.normal(e, w, std=1.0 / math.sqrt(w)),
                    bias=g.normal(e, std=0.05) if case["bias"] else None,
                    ids=torch.zeros(t, case["used"], dtype=torch.int32, device="cuda"),
                    weights=torch.zeros(t, case["used"], device="cuda"))
    if op == "product":
        e, r, c, p = case["experts"], case["rows"], case["cols"], case["pairs"]
        used = case["share"] if case["share"] > 1 else 1
        return dict(w=g.matrix(case["kind"], e * r, c), x=g.normal(p // case["share"], c),
                    ids=g.choice(p // used, e, min(used, e)).repeat(1, -(-used // e))[:, :used].reshape(-1).contiguous(),
                    y=torch.zeros(p, r, device="cuda"))
    if op == "mlp":
        e, w, h, t = case["experts"], case["width"], case["hidden"], case["tokens"]
        weights = torch.softmax(g.normal(t, case["used"]), 1)
        return dict(gate=g.matrix(case["kind"], e * h, w), up=g.matrix(case["kind"], e * h, w),
                    down=g.matrix(case["down"], e * w, h), x=g.normal(t, w), ids=g.choice(t, e, case["used"]),
                    weights=weights.contiguous(), out=torch.zeros(t, w, device="cuda"))
    t, kvw, qw = case["tokens"], case["kv_heads"] * case["head_dim"], case["heads"] * case["head_dim"]
    seqs, room = 1 if case["chunk"] else t, (case["length"] + 63) // 64 * 64
    return dict(q=g.normal(t, qw), kc=g.cache(case["form"], seqs * room, kvw), vc=g.cache(case["form"], seqs * room, kvw),
                index=g.order(seqs * room).reshape(seqs, room).contiguous() if case["paged"] else None,
                pos=torch.tensor(_ends(case), dtype=torch.int32, device="cuda"), room=room,
                out=torch.zeros(t, qw, device="cuda"))


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, _Inputs(seed)))
    if own:
        from molla_amd import gpu
        s["ctx"] = gpu.DeviceContext(0)
        for n, kind, cols in (("w", case.get("kind"), case.get("cols")), ("gate", case.get("kind"), case.get("width")),
                              ("up", case.get("kind"), case.get("width")), ("down", case.get("down"), case.get("hidden"))):
            if n in s:
                s["t_" + n] = gpu.Tensor(s[n].data_ptr(), kind, cols, s[n].shape[0], keep=s[n])
    return s


# ---- one pass --------------------------------------------------------------
def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def _own_router(s):
    from molla_amd import gpu
    c = s["case"]
    gpu.device_router(s["ctx"], s["x"], s["router"], s["ids"], s["weights"], bias=s["bias"], sigmoid=c["sigmoid"],
                      norm=c["norm"])
    return dict(ids=s["ids"], weights=s["weights"])


def _own_product(s):
    from molla_amd import gpu
    gpu.device_experts_matmul(s["ctx"], s["t_w"], s["case"]["experts"], s["x"], s["ids"], s["y"])
    return s["y"]


def _own_mlp(s):
    from molla_amd import gpu
    gpu.device_experts_mlp(s["ctx"], s["t_gate"], s["t_up"], s["t_down"], s["case"]["experts"], s["x"], s["ids"],
                           s["weights"], s["out"])
    return s["out"]


def _own_window(s):
    from molla_amd import gpu
    c = s["case"]
    gpu.device_attend_window(s["ctx"], s["q"], s["kc"], s["vc"], c["heads"], c["kv_heads"], c["head_dim"],
                             1.0 / math.sqrt(c["head_dim"]), c["window"], c["first"], s["pos"], c["length"], s["out"],
                             cache_stride=0 if c["chunk"] else s["room"] * s["kc"].shape[1],
                             kv_index=s["index"][0] if c["paged"] and c["chunk"] else s["index"],
                             form=gpu.CACHE_Q8 if c["form"] == Q8 else gpu.CACHE_F16)
    return s["out"]


def _plain_router(s):
    # (in 64 bits: which of two near scores is larger is a border)
    c, logits = s["case"], s["x"].double() @ s["router"].double().T
    p = torch.sigmoid(logits) if c["sigmoid"] else torch.softmax(logits, 1)
    score = p + s["bias"].double() if c["bias"] else p
    ids = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :c["used"]]
    w = p.gather(1, ids)
    w = w / w.sum(1, keepdim=True) if c["norm"] else w
    return dict(ids=ids.int(), weights=w.float())


def _halves(b):
    return b.contiguous().view(torch.float16).float()


def _values(kind, rows):
    """Weights of packed rows (n, bytes) in float32."""
    n, (_, size) = rows.shape[0], BLOCK[kind]
    b = rows.reshape(-1, size)
    if kind == Q8_0:
        v = _halves(b[:, :2]) * b[:, 2:].contiguous().view(torch.int8).float()
    elif kind == Q4_0:
        v = _halves(b[:, :2]) * (torch.cat([b[:, 2:] & 15, b[:, 2:] >> 4], 1).float() - 8.0)
    elif kind == Q4_K:
        d, s = _halves(b[:, :4]), b[:, 4:16]
        scale = torch.cat([s[:, :4] & 63, (s[:, 8:] & 15) | (s[:, :4] >> 6 << 4)], 1).float() * d[:, :1]
        least = torch.cat([s[:, 4:8] & 63, (s[:, 8:] >> 4) | (s[:, 4:8] >> 6 << 4)], 1).float() * d[:, 1:]
        q = b[:, 16:].reshape(-1, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], 2).reshape(-1, 8, 32).float()
        v = scale[:, :, None] * q - least[:, :, None]
    else:
        low, high = b[:, :128].reshape(-1, 2, 1, 64), b[:, 128:192].reshape(-1, 2, 1, 32)
        q = torch.cat([low & 15, low >> 4], 2).reshape(-1, 2, 4, 32)
        q = q | torch.cat([(high & 3) << 4, (high & 12) << 2, high & 48, (high & 192) >> 2], 2)
        scale = b[:, 192:208].contiguous().view(torch.int8).float() * _halves(b[:, 208:])
        v = (q.float() - 32.0).reshape(-1, 16, 16) * scale[:, :, None]
    return v.reshape(n, -1)


def _grouped(kind, w, experts, x, ids):
    """Row i of x against the matrix of expert ids[i]."""
    rows = w.shape[0] // experts
    w = w.reshape(experts, rows, -1)
    y = torch.zeros(x.shape[0], rows, device=x.device)
    if x.shape[0] <= 16:
        for i in range(x.shape[0]):
            y[i] = _values(kind, w.index_select(0, ids[i:i + 1].long())[0]) @ x[i]
        return y
    for e in range(experts):
        mine = (ids == e).nonzero()[:, 0]
        if mine.numel():
            y[mine] = x[mine] @ _values(kind, w[e]).T
    return y


def _plain_product(s):
    c = s["case"]
    return _grouped(c["kind"], s["w"], c["experts"], s["x"].repeat_interleave(c["share"], 0), s["ids"])


def _plain_mlp(s):
    c = s["case"]
    ids = s["ids"].reshape(-1)
    x = s["x"].repeat_interleave(c["used"], 0)
    gate = _grouped(c["kind"], s["gate"], c["experts"], x, ids)
    up = _grouped(c["kind"], s["up"], c["experts"], x, ids)
    y = _grouped(c["down"], s["down"], c["experts"], gate * torch.sigmoid(gate) * up, ids)
    return (y.reshape(c["tokens"], c["used"], -1) * s["weights"][:, :, None]).sum(1)


def _cached(s, cache, at, wide):
    """The cache's values at positions `at` (sequences, keys): (sequences, kv heads, keys, head_dim) in type `wide`."""
    c = s["case"]
    kvw = c["kv_heads"] * c["head_dim"]
    seqs, keys = at.shape
    cell = s["index"].gather(1, at).long() if c["paged"] else at + s["room"] * torch.arange(seqs, device=at.device)[:, None]
    rows = cache[cell.reshape(-1)]
    if c["form"] == F16:
        v = rows.to(wide)
    else:
        q = rows[:, :kvw // 2].contiguous().view(torch.int8).to(wide).reshape(-1, kvw // 32, 32)
        v = (q * rows[:, kvw // 2:kvw // 2 + kvw // 32].to(wide)[..., None]).reshape(-1, kvw)
    return v.reshape(seqs, keys, c["kv_heads"], c["head_dim"]).transpose(1, 2)


def _plain_window(s):
    c = s["case"]
    t, kvh, d = c["tokens"], c["kv_heads"], c["head_dim"]
    group, pos = c["heads"] // kvh, s["pos"].long()
    scale = 1.0 / math.sqrt(d)
    if c["chunk"]:  # every position up to the last, masked
        at = torch.arange(c["length"], device="cuda")[None]
        q = s["q"].reshape(1, t, kvh, group, d).permute(0, 2, 3, 1, 4).reshape(1, kvh, group * t, d)
        j, p = at[0], pos[:, None]
        seen = ((j <= p) & ((j > p - c["window"]) | (j < c["first"])))[None, None, None]
    else:  # the first positions and the window's, by sequence
        n = min(c["window"], c["length"])
        near = pos[:, None] - n + 1 + torch.arange(n, device="cuda")
        far = torch.arange(min(c["first"], c["length"]), device="cuda").expand(t, -1)
        seen = torch.cat([(far <= pos[:, None] - n) & (far <= pos[:, None]), near >= 0], 1)[:, None, None, None]
        at = torch.cat([far, near.clamp(min=0)], 1)
        q = s["q"].reshape(t, 1, kvh, group, d).permute(0, 2, 3, 1, 4).reshape(t, kvh, group, d)
    k, v = (_cached(s, cache, at, torch.float32).contiguous() for cache in (s["kc"], s["vc"]))
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    score = score.reshape(at.shape[0], kvh, group, -1, at.shape[1]).masked_fill(~seen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(p.reshape(at.shape[0], kvh, -1, at.shape[1]), v).reshape(at.shape[0], kvh, group, -1, d)
    o = o / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(t, -1)


_OWN = dict(router=_own_router, product=_own_product, mlp=_own_mlp, window=_own_window)
_PLAIN = dict(router=_plain_router, product=_plain_product, mlp=_plain_mlp, window=_plain_window)


# ---- what a pass cannot do without -----------------------------------------
def _touched(experts, tokens, used):
    """Experts that some token takes, on average and if all were as popular."""
    return max(min(used, experts), int(experts * (1.0 - (1.0 - min(used, experts) / experts) ** tokens)))


def _bytes(kind, values):
    per, size = BLOCK[kind]
    return values // per * size


def work(case):
    op = case["op"]
    if op == "router":
        t, w, e = case["tokens"], case["width"], case["experts"]
        return dict(bytes=4 * (t * w + e * w) + 8 * t * case["used"], flops=2 * t * w * e)
    if op == "product":
        r, c, p = case["rows"], case["cols"], case["pairs"]
        return dict(bytes=_touched(case["experts"], p // case["share"], case["share"]) * _bytes(case["kind"], r * c)
                    + 4 * p // case["share"] * c + 4 * p * r + 4 * p, flops=2 * p * r * c)
    if op == "mlp":
        w, h, p = case["width"], case["hidden"], case["tokens"] * case["used"]
        one = 2 * _bytes(case["kind"], w * h) + _bytes(case["down"], w * h)
        return dict(bytes=_touched(case["experts"], case["tokens"], case["used"]) * one + 8 * case["tokens"] * w + 8 * p, flops=6 * p * w * h)
    qw, kvw = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    cell = 2 * kvw if case["form"] == F16 else kvw + kvw // 16
    lows = [max(0, p + 1 - case["window"]) for p in _ends(case)]
    seen = [p + 1 - lo + min(case["first"], lo) for p, lo in zip(_ends(case), lows)]
    keys = case["length"] - lows[0] + min(case["first"], lows[0]) if case["chunk"] else sum(seen)
    return dict(bytes=2 * cell * keys + 8 * qw * case["tokens"], flops=4 * qw * sum(seen))


# ---- the same in 64 bits ---------------------------------------------------
def _half_bits(lo, hi):
    return (lo.to(torch.int32) | (hi.to(torch.int32) << 8)).to(torch.int16).view(torch.float16).double()


def _weight64(kind, rows):
    """Weights of packed rows (n, bytes) in float64, value by value of a block."""
    per, size = BLOCK[kind]
    b = rows.reshape(-1, size)
    v = torch.empty(b.shape[0], per, dtype=torch.float64, device=b.device)
    if kind in (Q8_0, Q4_0):
        d = _half_bits(b[:, 0], b[:, 1])
        for i in range(per):
            if kind == Q8_0:
                q = b[:, 2 + i].contiguous().view(torch.int8).double()
            else:
                q = ((b[:, 2 + i % 16] >> (4 * (i // 16))) & 15).double() - 8
            v[:, i] = q * d
    elif kind == Q4_K:
        d, dmin = _half_bits(b[:, 0], b[:, 1]), _half_bits(b[:, 2], b[:, 3])
        for j in range(8):
            if j < 4:
                sc, m = b[:, 4 + j] & 63, b[:, 8 + j] & 63
            else:
                sc = (b[:, 8 + j] & 15) | ((b[:, j] >> 6) << 4)
                m = (b[:, 8 + j] >> 4) | ((b[:, 4 + j] >> 6) << 4)
            q = (b[:, 16 + 32 * (j // 2):48 + 32 * (j // 2)] >> (4 * (j % 2))) & 15
            v[:, 32 * j:32 * j + 32] = q.double() * (d * sc.double())[:, None] - (dmin * m.double())[:, None]
    else:
        d = _half_bits(b[:, 208], b[:, 209])
        sc = b[:, 192:208].contiguous().view(torch.int8).double()
        for half in range(2):
            for part in range(4):
                lo = (b[:, 64 * half + 32 * (part % 2):64 * half + 32 * (part % 2) + 32] >> (4 * (part // 2))) & 15
                hi = (b[:, 128 + 32 * half:160 + 32 * half] >> (2 * part)) & 3
                q = (lo | (hi << 4)).double() - 32
                at = 128 * half + 32 * part
                v[:, at:at + 16] = q[:, :16] * (d * sc[:, 8 * half + 2 * part])[:, None]
                v[:, at + 16:at + 32] = q[:, 16:] * (d * sc[:, 8 * half + 2 * part + 1])[:, None]
    return v.reshape(rows.shape[0], -1)


def exact(case, seed):
    s = _inputs(case, _Inputs(seed))
    op = case["op"]
    if op == "router":
        logits = (s["router"].double() @ s["x"].double().T.contiguous()).T
        if case["sigmoid"]:
            p = 1.0 / (1.0 + torch.exp(-logits))
        else:
            p = torch.exp(logits - logits.max(1, keepdim=True).values)
            p = p / p.sum(1, keepdim=True)
        left = p + (s["bias"].double() if case["bias"] else 0.0)
        ids = []
        for _ in range(case["used"]):  # the largest that is left; the first of equals
            best = (left == left.max(1, keepdim=True).values).int().argmax(1, keepdim=True)
            ids.append(best)
            left = left.scatter(1, best, -math.inf)
        ids = torch.cat(ids, 1)
        w = torch.gather(p, 1, ids)
        return dict(ids=ids.int(), weights=w / w.sum(1, keepdim=True) if case["norm"] else w)
    if op == "product":
        e, r, share = case["experts"], case["rows"], case["share"]
        y = torch.zeros(case["pairs"], r, dtype=torch.float64, device="cuda")
        for i in range(e):
            mine = torch.where(s["ids"] == i)[0]
            if mine.numel():
                y[mine] = (_weight64(case["kind"], s["w"][i * r:(i + 1) * r]) @ s["x"][mine // share].double().T.contiguous()).T
        return y
    if op == "mlp":
        e, w, h = case["experts"], case["width"], case["hidden"]
        out = torch.zeros(case["tokens"], w, dtype=torch.float64, device="cuda")
        for i in range(e):
            token, place = torch.where(s["ids"] == i)
            if not token.numel():
                continue
            x = s["x"][token].double().T.contiguous()
            g = _weight64(case["kind"], s["gate"][i * h:(i + 1) * h]) @ x
            u = _weight64(case["kind"], s["up"][i * h:(i + 1) * h]) @ x
            y = _weight64(case["down"], s["down"][i * w:(i + 1) * w]) @ (g / (1.0 + torch.exp(-g)) * u)
            out.index_add_(0, token, (y * s["weights"][token, place].double()).T.contiguous())
        return out
    s["case"] = case
    t, d, group = case["tokens"], case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(t, case["heads"] * d, dtype=torch.float64, device="cuda")
    for lo in range(0, t, 64 if case["chunk"] else 1):  # a chunk's tokens in turns
        p = s["pos"][lo:lo + (64 if case["chunk"] else 1)].long()
        j = torch.arange(int(p.max()) + 1, device="cuda")
        j = j[(j < case["first"]) | (j > p.min() - case["window"])]
        hidden = (j > p[:, None]) | ((j <= p[:, None] - case["window"]) & (j >= case["first"]))
        row = j if case["chunk"] else j + lo * s["room"]
        if case["paged"]:
            row = s["index"][0 if case["chunk"] else lo, j].long()
        k, v = (_rows64(case, c[row]) for c in (s["kc"], s["vc"]))
        for x in range(case["heads"]):
            at = slice(x // group * d, (x // group + 1) * d)
            score = s["q"][lo:lo + p.numel(), x * d:(x + 1) * d].double() @ k[:, at].T.contiguous() / math.sqrt(d)
            out[lo:lo + p.numel(), x * d:(x + 1) * d] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v[:, at]
    return out


def _rows64(case, rows):
    """What cache rows stand for."""
    if case["form"] == F16:
        return rows.double()
    kvw = case["kv_heads"] * case["head_dim"]
    factor = rows[:, kvw // 2:kvw // 2 + kvw // 32].double().repeat_interleave(32, 1)
    return rows[:, :kvw // 2].contiguous().view(torch.int8).double() * factor
