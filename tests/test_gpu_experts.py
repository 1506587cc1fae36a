"""The router, products grouped by expert and the experts' MLP against the same
in float64 over the dequantized weights.

Products: the matrices' gate of 1e-5 of the largest output.  (An activation is
off by at most 2^-23 of its group's or its own size; about 64 roundings of
2^-25 of a partial sum, whose size is within four of the largest output's where
a kind takes a minimum off, are 8 * 4 * 2^-25 = 1e-6 of it as they mostly fall,
and a missing limb or half of an activation is 2^-16 or 2^-11.)  The MLP: that
gate's error of gate and up carried through the activation and the down
projection by absolute values, and the gate again.  Weights of the router: the
float64 value rounded once, 2^-24, and a float64 exponential.
"""

import numpy as np
import pytest
import torch

import oracle
from molla_amd import gpu, synth

pytestmark = pytest.mark.gpu

KINDS = [gpu.Q_Q4_0, gpu.Q_Q4_1, gpu.Q_Q5_0, gpu.Q_Q5_1, gpu.Q_Q8_0, gpu.Q_Q4_K, gpu.Q_Q5_K, gpu.Q_Q6_K]
GATE = 1e-5


def ctx():
    return gpu.DeviceContext(0)


def stack(kind, experts, rows, cols, seed):
    """(device tensor, float64 [experts, rows, cols])."""
    blob = synth.quant_tensor(kind, experts * rows, cols, seed)
    w = gpu.Tensor.from_bytes(blob, kind, cols, experts * rows)
    v = oracle.dequant(kind, blob.numpy(), experts * rows * cols).astype(np.float64)
    return w, torch.from_numpy(v).reshape(experts, rows, cols).cuda()


def grouped(w, x, ids):
    """Row p of x against w[ids[p]], in float64; rows without an expert are zero."""
    out = torch.zeros(len(ids), w.shape[1], dtype=torch.float64, device="cuda")
    for p, e in enumerate(ids.tolist()):
        if 0 <= e < w.shape[0]:
            out[p] = w[e] @ x[p].double()
    return out


def choice(tokens, experts, used, seed):
    g = torch.Generator().manual_seed(seed)
    liked = torch.randn(experts, generator=g)
    return (liked + torch.randn(tokens, experts, generator=g)).topk(used, 1).indices.int().cuda().contiguous()


def product(kind, experts, rows, cols, x, ids, share=1, w=None, seed=5):
    w, want = stack(kind, experts, rows, cols, seed) if w is None else w
    y = torch.full((ids.numel(), rows), 7.25, device="cuda")
    gpu.device_experts_matmul(ctx(), w, experts, x, ids, y)
    live = (ids >= 0) & (ids < experts)
    ref = grouped(want, x.repeat_interleave(share, 0), ids.cpu())
    assert (y[~live] == 7.25).all()
    if live.any():
        err = (y.double() - ref)[live].abs().max().item()
        assert err <= GATE * ref[live].abs().max().item(), err
    return y


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pairs", [3, 64, 65, 200])
def test_product_every_kind(kind, pairs):
    experts, rows, cols = 5, 96, 512
    ids = choice(pairs, experts, 1, pairs).reshape(-1)
    product(kind, experts, rows, cols, synth.normal(pairs * cols, 3, "cuda").view(pairs, cols), ids)


@pytest.mark.parametrize("kind,cols", [(gpu.Q_Q4_K, 256), (gpu.Q_Q4_K, 1024), (gpu.Q_Q4_K, 2304), (gpu.Q_Q4_K, 4352),
                                       (gpu.Q_Q6_K, 2048), (gpu.Q_Q6_K, 8448), (gpu.Q_Q8_0, 64), (gpu.Q_Q8_0, 320),
                                       (gpu.Q_Q5_1, 4160), (gpu.Q_Q4_0, 1088)])
@pytest.mark.parametrize("pairs", [1, 7, 90])
def test_product_widths_and_odd_rows(kind, cols, pairs):
    experts, rows = 3, 37
    ids = choice(pairs, experts, 1, cols + pairs).reshape(-1)
    product(kind, experts, rows, cols, synth.normal(pairs * cols, cols, "cuda").view(pairs, cols), ids)


@pytest.mark.parametrize("pairs", [12, 320])
def test_product_shared_rows(pairs):
    experts, rows, cols, share = 7, 64, 256, 4
    ids = choice(pairs // share, experts, share, 1).reshape(-1)
    product(gpu.Q_Q4_K, experts, rows, cols, synth.normal(pairs // share * cols, 1, "cuda").view(-1, cols), ids, share)


@pytest.mark.parametrize("pairs", [40, 300])
@pytest.mark.parametrize("case", ["one expert", "last expert", "none", "some not", "out of range", "ends"])
def test_product_unequal_shares(pairs, case):
    experts, rows, cols = 6, 160, 256
    ids = torch.randint(0, experts, (pairs,), generator=torch.Generator().manual_seed(2)).int()
    if case == "one expert":
        ids[:] = 2
    elif case == "last expert":
        ids[:] = experts - 1
    elif case == "none":
        ids[:] = -1
    elif case == "some not":
        ids[::3] = -1
    elif case == "out of range":
        ids[1::4] = experts
        ids[2::4] = 2**31 - 1
        ids[3::4] = -2**31
    else:
        ids[:] = 0
        ids[-1] = experts - 1
    product(gpu.Q_Q4_K, experts, rows, cols, synth.normal(pairs * cols, 4, "cuda").view(pairs, cols), ids.cuda())


def test_product_of_many_experts_and_large_counts():
    experts, rows, cols, pairs = 512, 32, 64, 3000
    ids = choice(pairs, experts, 1, 8).reshape(-1)
    product(gpu.Q_Q8_0, experts, rows, cols, synth.normal(pairs * cols, 4, "cuda").view(pairs, cols), ids)


@pytest.mark.parametrize("pairs", [8, 100])
def test_a_row_does_not_depend_on_the_others(pairs):
    """Infinities and NaN in one row, and the rows' order, change no bit of the others."""
    experts, rows, cols = 4, 128, 512
    w = stack(gpu.Q_Q4_K, experts, rows, cols, 9)
    x = synth.normal(pairs * cols, 4, "cuda").view(pairs, cols)
    ids = choice(pairs, experts, 1, 3).reshape(-1)
    y = product(gpu.Q_Q4_K, experts, rows, cols, x, ids, w=w)
    bad = x.clone()
    bad[3, 7], bad[5, 100] = float("nan"), float("inf")
    out = torch.zeros_like(y)
    gpu.device_experts_matmul(ctx(), w[0], experts, bad, ids, out)
    keep = [p for p in range(pairs) if p not in (3, 5)]
    assert torch.equal(out[keep], y[keep])
    turn = torch.randperm(pairs, generator=torch.Generator().manual_seed(1)).cuda()
    gpu.device_experts_matmul(ctx(), w[0], experts, x[turn].contiguous(), ids[turn].contiguous(), out)
    assert torch.equal(out, y[turn])


def mlp_reference(x, ids, weights, gate, up, down, act):
    """(out, bound) in float64."""
    tokens, used = ids.shape
    xr, flat = x.repeat_interleave(used, 0), ids.reshape(-1).cpu()
    g, u = grouped(gate, xr, flat), grouped(up, xr, flat)
    a = torch.nn.functional.gelu(g, approximate="tanh") if act else torch.nn.functional.silu(g)
    dh = GATE * (1.2 * g.abs().max() * u.abs() + a.abs() * u.abs().max()) + 2.0 ** -20 * (a * u).abs()
    y = grouped(down, a * u, flat)
    dy = grouped(down.abs(), dh, flat) + GATE * y.abs().max()
    w = weights.double()[..., None]
    return (w * y.view(tokens, used, -1)).sum(1), (w.abs() * dy.view(tokens, used, -1)).sum(1)




@pytest.mark.parametrize("kinds", [(gpu.Q_Q4_K, gpu.Q_Q6_K), (gpu.Q_Q8_0, gpu.Q_Q8_0), (gpu.Q_Q5_K, gpu.Q_Q4_K),
                                   (gpu.Q_Q4_0, gpu.Q_Q5_1), (gpu.Q_Q6_K, gpu.Q_Q4_0)])
@pytest.mark.parametrize("tokens,used", [(1, 2), (1, 6), (8, 4), (11, 6), (70, 2)])
@pytest.mark.parametrize("act,add", [(0, False), (gpu.ACT_BIT, True)])
def test_mlp(kinds, tokens, used, act, add):
    experts, width, hidden = 6, 256, 512
    (gate, g64), (up, u64) = (stack(kinds[0], experts, hidden, width, s) for s in (1, 2))
    down, d64 = stack(kinds[1], experts, width, hidden, 3)
    x = synth.normal(tokens * width, 6, "cuda", std=0.05).view(tokens, width)
    ids = choice(tokens, experts, used, tokens)
    weights = torch.rand(tokens, used, generator=torch.Generator().manual_seed(1)).cuda()
    out = synth.normal(tokens * width, 7, "cuda").view(tokens, width)
    held = out.clone().double()
    gpu.device_experts_mlp(ctx(), gate, up, down, experts, x, ids, weights, out, act, add)
    want, bound = mlp_reference(x, ids, weights, g64, u64, d64, act)
    if add:
        want = want + held
    assert ((out.double() - want).abs() <= bound + 2.0 ** -22 * want.abs()).all()


@pytest.mark.parametrize("tokens", [2, 40])
def test_mlp_pairs_without_an_expert(tokens):
    experts, width, hidden, used = 4, 256, 256, 3
    (gate, g64), (up, u64), (down, d64) = (stack(gpu.Q_Q4_K, experts, r, c, s) for r, c, s in
                                           ((hidden, width, 1), (hidden, width, 2), (width, hidden, 3)))
    x = synth.normal(tokens * width, 6, "cuda", std=0.05).view(tokens, width)
    ids = choice(tokens, experts, used, 5)
    ids[0] = -1                # a padded row
    ids[1, 1] = experts + 3
    ids[1, 2] = ids[1, 0]      # the same expert twice
    weights = torch.rand(tokens, used, generator=torch.Generator().manual_seed(1)).cuda()
    weights[1, 1] = float("nan")
    out = torch.full((tokens, width), 3.0, device="cuda")
    gpu.device_experts_mlp(ctx(), gate, up, down, experts, x, ids, weights, out)
    want, bound = mlp_reference(x, ids, torch.nan_to_num(weights), g64, u64, d64, 0)
    assert (out[0] == 0).all()
    assert ((out.double() - want).abs() <= bound).all()
    gpu.device_experts_mlp(ctx(), gate, up, down, experts, x, ids, weights, x)  # in place
    assert torch.equal(x, out)


def route_reference(x, router, bias, sigmoid, norm, used, scale):
    logits = x.double() @ router.double().T.contiguous()
    p = torch.sigmoid(logits) if sigmoid else torch.softmax(logits, 1)
    ids = torch.sort(p if bias is None else p + bias.double(), dim=1, descending=True, stable=True).indices[:, :used]
    w = p.gather(1, ids)
    return ids.int(), scale * (w / w.sum(1, keepdim=True) if norm else w)


@pytest.mark.parametrize("experts,used", [(1, 1), (8, 2), (60, 4), (64, 8), (65, 1), (128, 12), (160, 6), (512, 64)])
@pytest.mark.parametrize("tokens,width", [(1, 256), (3, 1028), (33, 64), (130, 512)])
@pytest.mark.parametrize("sigmoid,bias,norm", [(False, False, True), (True, True, True), (True, False, False),
                                               (False, True, False)])
def test_router(experts, used, tokens, width, sigmoid, bias, norm):
    x = synth.normal(tokens * width, 1, "cuda").view(tokens, width)
    router = synth.normal(experts * width, 2, "cuda", std=2.0 / width ** 0.5).view(experts, width)
    b = synth.normal(experts, 3, "cuda", std=0.02) if bias else None
    ids = torch.full((tokens, used), -5, dtype=torch.int32, device="cuda")
    weights = torch.zeros(tokens, used, device="cuda")
    gpu.device_router(ctx(), x, router, ids, weights, bias=b, sigmoid=sigmoid, norm=norm, scale=1.5)
    want, w = route_reference(x, router, b, sigmoid, norm, used, 1.5)
    assert torch.equal(ids, want)
    assert ((weights.double() - w).abs() <= 2.0 ** -23 * w).all()


def test_router_ties_go_low_and_far_logits():
    tokens, width, experts, used = 5, 128, 96, 7
    x = synth.normal(tokens * width, 1, "cuda").view(tokens, width)
    router = synth.normal(8 * width, 2, "cuda").view(8, width).repeat(12, 1).contiguous()  # equal by eights
    ids, weights = torch.zeros(tokens, used, dtype=torch.int32, device="cuda"), torch.zeros(tokens, used, device="cuda")
    gpu.device_router(ctx(), x, router, ids, weights)
    best = (x.double() @ router[:8].double().T).argmax(1).int()
    assert torch.equal(ids, best[:, None] + 8 * torch.arange(used, device="cuda", dtype=torch.int32))
    assert (weights - 1.0 / used).abs().max() <= 2.0 ** -24
    # logits of thousands: all but the largest weights are zero, and lowest ids fill the rest
    gpu.device_router(ctx(), 1e3 * x, router[:8].contiguous(), ids, weights)
    assert torch.equal(ids[:, 0], best) and (weights[:, 0] == 1).all()
    for row in ids.tolist():
        assert sorted(row) == sorted(set(row))


@pytest.mark.parametrize("sigmoid", [False, True])
def test_router_over_what_is_not_finite(sigmoid):
    """Ids stay experts, each once, whatever the values; other tokens do not change."""
    tokens, width, experts, used = 6, 64, 20, 5
    x = synth.normal(tokens * width, 1, "cuda").view(tokens, width)
    router = synth.normal(experts * width, 2, "cuda").view(experts, width)
    ids, weights = torch.zeros(tokens, used, dtype=torch.int32, device="cuda"), torch.zeros(tokens, used, device="cuda")
    gpu.device_router(ctx(), x, router, ids, weights, sigmoid=sigmoid)
    held, held_w = ids.clone(), weights.clone()
    x[1, 3], x[2, 5], x[4] = float("nan"), float("inf"), -float("inf")
    gpu.device_router(ctx(), x, router, ids, weights, sigmoid=sigmoid)
    assert torch.equal(ids[[0, 3, 5]], held[[0, 3, 5]]) and torch.equal(weights[[0, 3, 5]], held_w[[0, 3, 5]])
    for row in ids.tolist():
        assert len(set(row)) == used and all(0 <= e < experts for e in row)
    if not sigmoid:
        assert ids[1].tolist() == list(range(used))


def test_captured_and_replayed():
    """Router and MLP in one graph, replayed over new inputs with eager work between."""
    tokens, experts, used, width, hidden = 8, 8, 2, 256, 256
    s = torch.cuda.Stream()
    c = gpu.DeviceContext(0, s)
    (gate, _), (up, _), (down, _) = (stack(gpu.Q_Q4_K, experts, r, k, n) for r, k, n in
                                     ((hidden, width, 1), (hidden, width, 2), (width, hidden, 3)))
    router = synth.normal(experts * width, 4, "cuda").view(experts, width)
    big = synth.normal(40 * width, 9, "cuda").view(40, width)
    for x in (big[:tokens].contiguous(), big):
        n = x.shape[0]
        ids, weights = torch.zeros(n, used, dtype=torch.int32, device="cuda"), torch.zeros(n, used, device="cuda")
        out = torch.zeros(n, width, device="cuda")
        torch.cuda.synchronize()

        def step():
            gpu.device_router(c, x, router, ids, weights)
            gpu.device_experts_mlp(c, gate, up, down, experts, x, ids, weights, out)

        c.workspace(64 << 20)
        with torch.cuda.stream(s):
            step()
            c.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step()
        for k in range(4):
            with torch.cuda.stream(s):
                x.copy_(synth.normal(n * width, 20 + k, "cuda").view(n, width))
                g.replay()
                got = out.clone()
                out.zero_()
                step()
            c.synchronize()
            assert torch.equal(got, out) and out.abs().max() > 0
