"""Products of many rows with stacked experts' matrices at every width of block
that they are cut into, the experts' MLP with its down projection's columns in
parts, both sides of the rules that choose, and calls beside each other.

Gates as tests/test_gpu_experts.py derives them: a product within 1e-5 of the
largest output, the MLP within that carried through by absolute values.
"""

import numpy as np
import pytest
import torch

import oracle
from molla_amd import MiError, gpu, synth

pytestmark = pytest.mark.gpu

KINDS = [gpu.Q_Q4_0, gpu.Q_Q4_1, gpu.Q_Q5_0, gpu.Q_Q5_1, gpu.Q_Q8_0, gpu.Q_Q4_K, gpu.Q_Q5_K, gpu.Q_Q6_K]
GATE = 1e-5
# rows of each expert, so that a block holds 1, 2 or 4 tiles of 32 of them, and what
# is left behind whole blocks 1 to 4 tiles, full ones and not
SHARES = {"two": (10, 40, 70, 30, 0, 64), "two or four": (100, 40, 70, 150, 65, 128), "four": (33, 97, 257, 1, 130, 160)}


def stack(kind, experts, rows, cols, seed):
    """(device tensor, float64 [experts, rows, cols])."""
    blob = synth.quant_tensor(kind, experts * rows, cols, seed)
    w = gpu.Tensor.from_bytes(blob, kind, cols, experts * rows)
    v = oracle.dequant(kind, blob.numpy(), experts * rows * cols).astype(np.float64)
    return w, torch.from_numpy(v).reshape(experts, rows, cols).cuda()


def grouped(w, x, ids):
    """Row p of x against w[ids[p]] in float64; rows without an expert are zero."""
    out = torch.zeros(len(ids), w.shape[1], dtype=torch.float64, device="cuda")
    for e in range(w.shape[0]):
        at = (ids == e).nonzero()[:, 0]
        if len(at):
            out[at] = x[at].double() @ w[e].T.contiguous()
    return out


def shares(which, seed):
    ids = torch.tensor([e for e, n in enumerate(SHARES[which]) for _ in range(n)], dtype=torch.int32)
    return ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(seed))].cuda()


def held(y, want):
    return (y.double() - want).abs().max().item() <= GATE * want.abs().max().item()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("which", list(SHARES))
@pytest.mark.parametrize("rows,cols", [(200, 512), (384, 768), (37, 1280)])
def test_product_by_shares(kind, which, rows, cols):
    w, w64 = stack(kind, 6, rows, cols, 5)
    ids = shares(which, rows)
    x = synth.normal(len(ids) * cols, 3, "cuda").view(-1, cols)
    y = torch.full((len(ids), rows), 7.25, device="cuda")
    gpu.device_experts_matmul(gpu.DeviceContext(0), w, 6, x, ids, y)
    assert held(y, grouped(w64, x, ids))


def mlp(kinds, experts, width, hidden, x, ids, weights, act=0, onto=None, work=None, c=None):
    """The MLP's output, checked against float64."""
    (gate, g64), (up, u64) = (stack(kinds[0], experts, hidden, width, s) for s in (1, 2))
    down, d64 = stack(kinds[1], experts, width, hidden, 3)
    out = torch.zeros_like(x) if onto is None else onto.clone()
    gpu.device_experts_mlp(c or gpu.DeviceContext(0), gate, up, down, experts, x, ids, weights, out, act, onto is not None,
                           work=work)
    tokens, used = ids.shape
    flat, xr = ids.reshape(-1), x.repeat_interleave(used, 0)
    g, u = grouped(g64, xr, flat), grouped(u64, xr, flat)
    a = torch.nn.functional.gelu(g, approximate="tanh") if act else torch.nn.functional.silu(g)
    dh = GATE * (1.2 * g.abs().max() * u.abs() + a.abs() * u.abs().max()) + 2.0 ** -20 * (a * u).abs()
    y = grouped(d64, a * u, flat)
    dy = grouped(d64.abs(), dh, flat) + GATE * y.abs().max()
    wt = weights.double()[..., None]
    want, bound = (wt * y.view(tokens, used, -1)).sum(1), (wt.abs() * dy.view(tokens, used, -1)).sum(1)
    if onto is not None:
        want = want + onto.double()
    assert ((out.double() - want).abs() <= bound + 2.0 ** -22 * want.abs()).all()
    return out


@pytest.mark.parametrize("kinds", [(k, KINDS[-1 - n]) for n, k in enumerate(KINDS)])
@pytest.mark.parametrize("which", list(SHARES))
def test_mlp_by_shares(kinds, which):
    """Every kind as gate and up and as down, hidden rows no whole number of blocks."""
    ids = shares(which, 7).view(-1, 1)
    x = synth.normal(len(ids) * 256, 6, "cuda", std=0.05).view(-1, 256)
    weights = torch.rand(len(ids), 1, generator=torch.Generator().manual_seed(1)).cuda()
    mlp(kinds, 6, 256, 768, x, ids, weights, gpu.ACT_BIT if which == "two" else 0)


@pytest.mark.parametrize("kind", [gpu.Q_Q4_K, gpu.Q_Q6_K, gpu.Q_Q8_0])
@pytest.mark.parametrize("hidden,tokens", [(4096, 40), (4352, 40), (8192, 33), (8448, 100), (16640, 45)])
def test_mlp_with_columns_in_parts(kind, hidden, tokens):
    """Down projections of few blocks: their columns in two, four and eight parts, equal and not."""
    used, width = 2, 256
    g = torch.Generator().manual_seed(tokens)
    ids = torch.stack([torch.randperm(3, generator=g)[:used] for _ in range(tokens)]).int().cuda()
    ids[5, 1] = -1
    x = synth.normal(tokens * width, 6, "cuda", std=0.05).view(tokens, width)
    weights = torch.rand(tokens, used, generator=g).cuda()
    onto = synth.normal(tokens * width, 8, "cuda").view(tokens, width)
    mlp((gpu.Q_Q4_K, kind), 3, width, hidden, x, ids, weights)
    mlp((gpu.Q_Q4_K, kind), 3, width, hidden, x, ids, weights, onto=onto)


@pytest.mark.parametrize("experts,pairs,rows,cols", [(4, 12, 2048, 1024), (4, 23, 2048, 1024), (4, 25, 2048, 1024),
                                                     (2, 64, 1024, 768), (2, 64, 1024, 512), (30, 64, 256, 256),
                                                     (30, 65, 256, 256)])
def test_both_sides_of_few(experts, pairs, rows, cols):
    w, w64 = stack(gpu.Q_Q4_K, experts, rows, cols, 5)
    ids = torch.randint(0, experts, (pairs,), generator=torch.Generator().manual_seed(2)).int().cuda()
    x = synth.normal(pairs * cols, 3, "cuda").view(pairs, cols)
    y = torch.full((pairs, rows), 7.25, device="cuda")
    gpu.device_experts_matmul(gpu.DeviceContext(0), w, experts, x, ids, y)
    assert held(y, grouped(w64, x, ids))


@pytest.mark.parametrize("tokens,used,experts", [(1, 2, 4), (7, 3, 4), (20, 2, 40), (33, 2, 4), (150, 3, 4)])
def test_exact_workspaces(tokens, used, experts):
    """Each call on exactly its workspace, among bytes that stay as they were; less is refused."""
    width, hidden, kind = 256, 4352, gpu.Q_Q4_K
    c, L = gpu.DeviceContext(0), gpu.lib()
    g = torch.Generator().manual_seed(4)
    ids = torch.stack([torch.randperm(experts, generator=g)[:used] for _ in range(tokens)]).int().cuda()
    x = synth.normal(tokens * width, 6, "cuda", std=0.05).view(tokens, width)
    weights = torch.rand(tokens, used, generator=g).cuda()
    gate, up = (stack(kind, experts, hidden, width, s)[0] for s in (1, 2))
    down = stack(kind, experts, width, hidden, 3)[0]
    router = synth.normal(experts * width, 4, "cuda").view(experts, width)
    y, out = torch.zeros(tokens * used, hidden, device="cuda"), torch.zeros(tokens, width, device="cuda")
    d = gpu.MiExperts(experts, width, hidden, 0, gate.weight(), up.weight(), down.weight())
    picks, parts = torch.zeros_like(ids), torch.zeros_like(weights)
    calls = [(L.mi_experts_matmul_workspace(experts, width, used, tokens * used), y,
              lambda work: gpu.device_experts_matmul(c, gate, experts, x, ids, y, work=work)),
             (L.mi_experts_workspace(d, tokens, used), out,
              lambda work: gpu.device_experts_mlp(c, gate, up, down, experts, x, ids, weights, out, work=work)),
             (L.mi_router_workspace(experts, tokens), parts,
              lambda work: gpu.device_router(c, x, router, picks, parts, work=work))]
    for need, result, call in calls:
        call(None)
        want = result.clone()
        result.zero_()
        room = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
        call(room[256:256 + need])
        torch.cuda.synchronize()
        assert torch.equal(result, want)
        assert (room[:256] == 77).all() and (room[256 + need:] == 77).all()
        with pytest.raises(MiError):
            call(room[256:256 + need - 256])


@pytest.mark.parametrize("tokens", [1, 12, 90])
def test_two_contexts_at_once(tokens):
    """Two streams with a context each, their calls between one another's, as one after the other."""
    experts, used, width, hidden = 6, 2, 512, 1024
    (gate, _), (up, _), (down, _) = (stack(gpu.Q_Q4_K, experts, r, k, n) for r, k, n in
                                     ((hidden, width, 1), (hidden, width, 2), (width, hidden, 3)))
    router = synth.normal(experts * width, 4, "cuda").view(experts, width)
    runs = []
    for s in range(2):
        stream = torch.cuda.Stream()
        runs.append((gpu.DeviceContext(0, stream), synth.normal(tokens * width, 10 + s, "cuda").view(tokens, width),
                     torch.zeros(tokens, used, dtype=torch.int32, device="cuda"),
                     torch.zeros(tokens, used, device="cuda"), torch.zeros(8, tokens, width, device="cuda")))
    torch.cuda.synchronize()

    def step(run, k):
        c, x, ids, weights, out = run
        gpu.device_router(c, x, router, ids, weights)
        gpu.device_experts_mlp(c, gate, up, down, experts, x, ids, weights, out[k])

    for k in range(8):
        for run in runs:
            step(run, k)
    torch.cuda.synchronize()
    for run in runs:
        got = run[4].clone()
        run[4].zero_()
        torch.cuda.synchronize()
        step(run, 0)
        torch.cuda.synchronize()
        assert run[4][0].abs().max() > 0
        assert all(torch.equal(got[k], run[4][0]) for k in range(8))


def test_another_stream_than_the_tensors():
    """Inputs made on the default stream, the call on a context's own, which waits for them."""
    experts, used, width, hidden, tokens = 4, 2, 256, 512, 40
    ids = torch.randint(0, experts, (tokens, used), generator=torch.Generator().manual_seed(2)).int().cuda()
    x = synth.normal(tokens * width, 6, "cuda", std=0.05).view(tokens, width)
    weights = torch.rand(tokens, used, generator=torch.Generator().manual_seed(1)).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    kinds = (gpu.Q_Q5_1, gpu.Q_Q5_0)
    with torch.cuda.stream(stream):
        a = mlp(kinds, experts, width, hidden, x, ids, weights, c=gpu.DeviceContext(0, stream))
    stream.synchronize()
    assert torch.equal(a, mlp(kinds, experts, width, hidden, x, ids, weights))
