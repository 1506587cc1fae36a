"""Products and MLPs of a few rows an expert on the matrix cores (Q4_K and Q6_K,
about 1.5 to 8 rows an expert), against float64.

Gates as tests/test_gpu_experts.py derives them.
"""

import numpy as np
import pytest
import torch

import oracle
from molla_amd import gpu, synth

pytestmark = pytest.mark.gpu

GATE = 1e-5


def stack(kind, experts, rows, cols, seed):
    """(device tensor, float64 [experts, rows, cols])."""
    blob = synth.quant_tensor(kind, experts * rows, cols, seed)
    w = gpu.Tensor.from_bytes(blob, kind, cols, experts * rows)
    v = oracle.dequant(kind, blob.numpy(), experts * rows * cols).astype(np.float64)
    return w, torch.from_numpy(v).reshape(experts, rows, cols).cuda()


def grouped(w, x, ids):
    out = torch.zeros(len(ids), w.shape[1], dtype=torch.float64, device="cuda")
    for e in range(w.shape[0]):
        at = (ids == e).nonzero()[:, 0]
        if len(at):
            out[at] = x[at].double() @ w[e].T.contiguous()
    return out


def product(kind, w, w64, x, ids, share=1):
    y = torch.full((ids.numel(), w64.shape[1]), 7.25, device="cuda")
    gpu.device_experts_matmul(gpu.DeviceContext(0), w, w64.shape[0], x, ids, y)
    want = grouped(w64, x.repeat_interleave(share, 0), ids.reshape(-1))
    live = ((ids >= 0) & (ids < w64.shape[0])).reshape(-1)
    assert (y[~live] == 7.25).all()
    assert (y.double() - want)[live].abs().max() <= GATE * want.abs().max()
    return y


def pattern(counts, seed):
    ids = torch.tensor([e for e, n in enumerate(counts) for _ in range(n)], dtype=torch.int32)
    return ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(seed))].cuda()


@pytest.mark.parametrize("kind", [gpu.Q_Q4_K, gpu.Q_Q6_K])
@pytest.mark.parametrize("rows,cols", [(37, 256), (128, 512), (200, 768), (129, 2304), (31, 8448), (300, 4096)])
@pytest.mark.parametrize("counts", [(1, 2, 8, 4), (3, 9, 0, 5), (17, 0, 0, 0), (0, 0, 8, 8), (5, 4, 3, 7)])
def test_product(kind, rows, cols, counts):
    w, w64 = stack(kind, 4, rows, cols, 5)
    ids = pattern(counts, rows)
    product(kind, w, w64, synth.normal(len(ids) * cols, 3, "cuda").view(-1, cols), ids)


@pytest.mark.parametrize("kind", [gpu.Q_Q4_K, gpu.Q_Q6_K])
def test_rows_of_very_different_sizes_and_columns_too(kind):
    """A row's scale is its own, by runs of 512 columns: each row to the gate of its own largest output."""
    experts, rows, cols, pairs = 3, 96, 2048, 10
    w, w64 = stack(kind, experts, rows, cols, 5)
    ids = pattern((3, 4, 3), 1)
    x = synth.normal(pairs * cols, 3, "cuda").view(pairs, cols)
    x *= torch.tensor([10.0 ** (4 * (p % 5) - 8) for p in range(pairs)], device="cuda")[:, None]
    x[:, :512] *= 1e-6
    x[2] = 0
    x[4, 512:] = 0
    y = product(kind, w, w64, x, ids)
    want = grouped(w64, x, ids)
    assert (y[2] == 0).all()
    assert ((y.double() - want).abs().amax(1) <= GATE * want.abs().amax(1)).all()


@pytest.mark.parametrize("kind", [gpu.Q_Q4_K, gpu.Q_Q6_K])
def test_shared_rows_and_pairs_without_an_expert(kind):
    experts, rows, cols, share = 4, 96, 512, 3
    w, w64 = stack(kind, experts, rows, cols, 9)
    ids = torch.tensor([[0, 1, 2], [1, 1, 3], [-1, 2, 0], [3, 4, 2], [2, -2**31, 1], [0, 1, 2**31 - 1]],
                       dtype=torch.int32, device="cuda").reshape(-1)
    product(kind, w, w64, synth.normal(6 * cols, 2, "cuda").view(6, cols), ids, share)
    none = torch.full((18,), -1, dtype=torch.int32, device="cuda")
    y = torch.full((18, rows), 7.25, device="cuda")
    gpu.device_experts_matmul(gpu.DeviceContext(0), w, experts, synth.normal(6 * cols, 2, "cuda").view(6, cols), none, y)
    assert (y == 7.25).all()


@pytest.mark.parametrize("kind", [gpu.Q_Q4_K, gpu.Q_Q6_K])
def test_a_row_does_not_depend_on_the_others(kind):
    experts, rows, cols, pairs = 3, 128, 1280, 12
    w, w64 = stack(kind, experts, rows, cols, 9)
    x = synth.normal(pairs * cols, 4, "cuda").view(pairs, cols)
    ids = pattern((9, 2, 1), 3)
    y = product(kind, w, w64, x, ids)
    bad = x.clone()
    bad[3, 7], bad[5, 1100], bad[8] = float("nan"), float("inf"), -float("inf")
    out = torch.zeros_like(y)
    c = gpu.DeviceContext(0)
    gpu.device_experts_matmul(c, w, experts, bad, ids, out)
    keep = [p for p in range(pairs) if p not in (3, 5, 8)]
    assert torch.equal(out[keep], y[keep])
    assert not torch.isfinite(out[[3, 5, 8]]).any()
    turn = torch.randperm(pairs, generator=torch.Generator().manual_seed(1)).cuda()
    gpu.device_experts_matmul(c, w, experts, x[turn].contiguous(), ids[turn].contiguous(), out)
    assert torch.equal(out, y[turn])


@pytest.mark.parametrize("kinds", [(gpu.Q_Q4_K, gpu.Q_Q4_K), (gpu.Q_Q4_K, gpu.Q_Q6_K), (gpu.Q_Q6_K, gpu.Q_Q4_K),
                                   (gpu.Q_Q6_K, gpu.Q_Q6_K)])
@pytest.mark.parametrize("width,hidden", [(256, 512), (512, 8448), (768, 1280)])
@pytest.mark.parametrize("tokens,used,experts", [(4, 3, 3), (6, 2, 4), (9, 2, 4), (8, 8, 16)])
@pytest.mark.parametrize("act,add", [(0, False), (gpu.ACT_BIT, True)])
def test_mlp(kinds, width, hidden, tokens, used, experts, act, add):
    """With a down projection's columns in up to eight parts, which the sum adds."""
    (gate, g64), (up, u64) = (stack(kinds[0], experts, hidden, width, s) for s in (1, 2))
    down, d64 = stack(kinds[1], experts, width, hidden, 3)
    g = torch.Generator().manual_seed(tokens)
    ids = torch.stack([torch.randperm(experts, generator=g)[:used] for _ in range(tokens)]).int().cuda()
    ids[1, 0] = -1
    x = synth.normal(tokens * width, 6, "cuda", std=0.05).view(tokens, width)
    weights = torch.rand(tokens, used, generator=g).cuda()
    out = synth.normal(tokens * width, 7, "cuda").view(tokens, width)
    held = out.double()
    gpu.device_experts_mlp(gpu.DeviceContext(0), gate, up, down, experts, x, ids, weights, out, act, add)
    flat, xr = ids.reshape(-1), x.repeat_interleave(used, 0)
    gt, ut = grouped(g64, xr, flat), grouped(u64, xr, flat)
    a = torch.nn.functional.gelu(gt, approximate="tanh") if act else torch.nn.functional.silu(gt)
    dh = GATE * (1.2 * gt.abs().max() * ut.abs() + a.abs() * ut.abs().max()) + 2.0 ** -20 * (a * ut).abs()
    y = grouped(d64, a * ut, flat)
    dy = grouped(d64.abs(), dh, flat) + GATE * y.abs().max()
    wt = weights.double()[..., None]
    want, bound = (wt * y.view(tokens, used, -1)).sum(1), (wt.abs() * dy.view(tokens, used, -1)).sum(1)
    if add:
        want = want + held
    assert ((out.double() - want).abs() <= bound + 2.0 ** -22 * want.abs()).all()
    if not add:
        gpu.device_experts_mlp(gpu.DeviceContext(0), gate, up, down, experts, x, ids, weights, x, act)  # in place
        assert torch.equal(x, out)


def test_captured_and_replayed():
    experts, used, width, hidden, tokens = 4, 2, 256, 4352, 6
    s = torch.cuda.Stream()
    c = gpu.DeviceContext(0, s)
    (gate, _), (up, _), (down, _) = (stack(gpu.Q_Q4_K, experts, r, k, n) for r, k, n in
                                     ((hidden, width, 1), (hidden, width, 2), (width, hidden, 3)))
    ids = torch.zeros(tokens, used, dtype=torch.int32, device="cuda")
    x, weights = torch.zeros(tokens, width, device="cuda"), torch.rand(tokens, used, device="cuda")
    out = torch.zeros(tokens, width, device="cuda")
    c.workspace(16 << 20)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        gpu.device_experts_mlp(c, gate, up, down, experts, x, ids, weights, out)
        c.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            gpu.device_experts_mlp(c, gate, up, down, experts, x, ids, weights, out)
    for k in range(4):
        with torch.cuda.stream(s):
            x.copy_(synth.normal(tokens * width, 20 + k, "cuda").view(tokens, width))
            ids.copy_(torch.randint(-1, experts, (tokens, used), generator=torch.Generator().manual_seed(k)))
            g.replay()
            got = out.clone()
            out.zero_()
            gpu.device_experts_mlp(c, gate, up, down, experts, x, ids, weights, out)
        c.synchronize()
        assert torch.equal(got, out) and out.abs().max() > 0
