"""Sparse experts and windowed attention at the ends of what the header allows:
the most tokens and pairs, matrices past 32 bits, running maxima that stay and move,
one cell many times.

Gates as tests/test_gpu_experts.py and tests/test_gpu_window.py derive them; a
windowed chunk's weights are, besides, each off by 2^-36 of the largest, which over n
positions is n 2^-36 of the largest value.
"""

import math

import numpy as np
import pytest
import torch

import oracle
from molla_amd import gpu, synth

pytestmark = pytest.mark.gpu

GATE = 1e-5


def dense(kind, blob, rows, cols):
    return torch.from_numpy(oracle.dequant(kind, blob.numpy(), rows * cols).astype(np.float64)).view(rows, cols).cuda()


def test_most_tokens():
    """65536 tokens: the router, the MLP over every way and its sum."""
    tokens, width, experts, used = 65536, 64, 3, 2
    c = gpu.DeviceContext(0)
    x = synth.normal(tokens * width, 1, "cuda").view(tokens, width)
    router = synth.normal(experts * width, 2, "cuda").view(experts, width)
    ids, weights = torch.zeros(tokens, used, dtype=torch.int32, device="cuda"), torch.zeros(tokens, used, device="cuda")
    gpu.device_router(c, x, router, ids, weights)
    p = torch.softmax(x.double() @ router.double().T.contiguous(), 1)
    want = torch.sort(p, dim=1, descending=True, stable=True)
    assert torch.equal(ids, want.indices[:, :used].int())
    blobs = [synth.quant_tensor(gpu.Q_Q8_0, experts * 64, 64, s) for s in (1, 2, 3)]
    gate, up, down = (gpu.Tensor.from_bytes(b, gpu.Q_Q8_0, 64, experts * 64) for b in blobs)
    g64, u64, d64 = (dense(gpu.Q_Q8_0, b, experts * 64, 64).view(experts, 64, 64) for b in blobs)
    out = torch.zeros(tokens, width, device="cuda")
    gpu.device_experts_mlp(c, gate, up, down, experts, x, ids, weights, out)
    for t in (0, 1, 31, 32, 4095, 32768, 65535):
        ref = sum(weights[t, k].double() * (d64[e] @ (torch.nn.functional.silu(g64[e] @ x[t].double()) * (u64[e] @ x[t].double())))
                  for k, e in enumerate(ids[t].tolist()))
        assert (out[t].double() - ref).abs().max() <= 1e-4 * ref.abs().max()


def test_most_pairs():
    pairs, rows, cols, experts = 1 << 20, 32, 64, 5
    blob = synth.quant_tensor(gpu.Q_Q4_0, experts * rows, cols, 1)
    w, w64 = gpu.Tensor.from_bytes(blob, gpu.Q_Q4_0, cols, experts * rows), dense(gpu.Q_Q4_0, blob, experts * rows, cols)
    x = synth.normal(pairs // 16 * cols, 1, "cuda").view(-1, cols)
    ids = torch.randint(0, experts, (pairs,), generator=torch.Generator().manual_seed(2)).int().cuda()
    y = torch.zeros(pairs, rows, device="cuda")
    gpu.device_experts_matmul(gpu.DeviceContext(0), w, experts, x, ids, y)
    at = torch.tensor([0, 1, 15, 16, 77777, 524288, pairs - 1], device="cuda")
    want = (w64.view(experts, rows, cols)[ids[at].long()] * x[at // 16].double()[:, None]).sum(2)
    assert (y[at].double() - want).abs().max() <= GATE * want.abs().max()
    assert (y != 0).any(1).all()


@pytest.mark.parametrize("kind,pairs", [(gpu.Q_Q8_0, 3), (gpu.Q_Q4_K, 120), (gpu.Q_Q4_K, 64), (gpu.Q_Q6_K, 400)])
def test_matrices_past_32_bits(kind, pairs):
    """A stack of more than 2^32 bytes: the first and the last expert, the others zeros."""
    rows, cols = 8192, 8192
    one = synth.quant_tensor(kind, rows, cols, 3, device="cuda")
    experts = (1 << 32) // one.numel() + 2
    if kind == gpu.Q_Q4_K and pairs == 64:
        experts = 34  # (two pairs an expert on average: the packed product)
        rows = -(-(1 << 32) // (33 * 4608))
        one = synth.quant_tensor(kind, rows, cols, 3, device="cuda")
    blob = torch.zeros(experts * one.numel(), dtype=torch.uint8, device="cuda")
    blob[:one.numel()] = one
    blob[-one.numel():] = one
    assert (experts - 1) * one.numel() >= 1 << 32
    w = gpu.Tensor.from_bytes(blob, kind, cols, experts * rows)
    ids = torch.full((pairs,), experts - 1, dtype=torch.int32, device="cuda")
    ids[::3] = 0
    x = synth.normal(pairs * cols, 1, "cuda").view(pairs, cols)
    y = torch.zeros(pairs, rows, device="cuda")
    gpu.device_experts_matmul(gpu.DeviceContext(0), w, experts, x, ids, y)
    some = 64
    w64 = dense(kind, one[:some * w.row_bytes()].cpu(), some, cols)
    want = x.double() @ w64.T.contiguous()
    assert (y[:, :some].double() - want).abs().max() <= GATE * want.abs().max()
    w64 = dense(kind, one[-some * w.row_bytes():].cpu(), some, cols)
    want = x.double() @ w64.T.contiguous()
    assert (y[:, -some:].double() - want).abs().max() <= GATE * want.abs().max()


def chunk(k, v, q, heads, kvh, d, scale, window, first, start, index=None):
    n = q.shape[0]
    pos = torch.arange(start, start + n, dtype=torch.int32, device="cuda")
    out = torch.zeros(n, heads * d, device="cuda")
    gpu.device_attend_window(gpu.DeviceContext(0), q, k, v, heads, kvh, d, scale, window, first, pos, start + n, out,
                             kv_index=index)
    j = torch.arange(start + n, device="cuda")
    seen = (j <= pos[:, None]) & ((j > pos[:, None] - window) | (j < first))
    at = j if index is None else index[:start + n].long()
    kk, vv = (x[at].double().view(-1, kvh, d).transpose(0, 1).contiguous() for x in (k, v))
    qq = q.double().view(n, kvh, -1, d).permute(1, 2, 0, 3).contiguous()  # [kvh, group, n, d]
    s = torch.matmul(qq, kk.transpose(1, 2).contiguous()[:, None]) * scale
    s = s.masked_fill(~seen, -math.inf)
    want = torch.matmul(torch.softmax(s, -1), vv[:, None]).permute(2, 0, 1, 3).reshape(n, heads * d)
    size = (torch.matmul(qq.abs(), kk.abs().transpose(1, 2).contiguous()[:, None]) * abs(scale)).max().item()
    reach = int(seen.sum(1).max())
    bound = vv.abs().max().item() * (2.0 ** -24 * (2 * (3 * d / 16 + 16) * size + reach / 8 + 64) + 2.0 ** -36 * reach)
    assert (out.double() - want).abs().max().item() <= bound
    return out


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("step", [0.002, 0.02, 0.2, -0.02, 0.0])
def test_scores_that_rise_and_fall(d, step):
    """Scores that grow by `step` a position, so that a row's maximum passes the one it
    holds by less than the factor that moves it, again and again, or never does."""
    n, start, heads, kvh = 70, 900, 4, 2
    g = torch.Generator().manual_seed(d)
    k, v = (torch.randn(start + n, kvh * d, generator=g) for _ in range(2))
    k = 0.05 * k
    k[:, ::d] = (torch.arange(start + n) * step)[:, None]
    q = torch.randn(n, heads * d, generator=g)
    q[:, ::d] = 1.0
    chunk(k.half().cuda(), v.half().cuda(), q.cuda(), heads, kvh, d, 1.0, 700, 9, start)
    chunk(k.half().cuda(), v.half().cuda(), q.cuda(), heads, kvh, d, -1.0, 700, 9, start)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [0.0, 1e-38, -1e-30, 1e-12])
def test_weights_that_are_all_equal(d, scale):
    n, start, heads, kvh = 40, 3000, 2, 1
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(start + n, kvh * d, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(n, heads * d, generator=g).cuda()
    chunk(k, v, q, heads, kvh, d, scale, 2500, 4, start)


@pytest.mark.parametrize("d", [64, 128])
def test_one_large_weight_over_many_small_ones(d):
    """A first position's weight 2^12 times each of 4000 others', which together outweigh
    half of it: ones that a row's later maximum must not round away."""
    n, start, heads, kvh = 33, 4100, 2, 1
    g = torch.Generator().manual_seed(6)
    k = torch.zeros(start + n, kvh * d)
    k[0, 0] = 12 * math.log(2.0)
    v = torch.randn(start + n, kvh * d, generator=g)
    v[1:] = v[1:].abs()
    q = torch.zeros(n, heads * d)
    q[:, ::d] = 1.0
    chunk(k.half().cuda(), v.half().cuda(), q.cuda(), heads, kvh, d, 1.0, 4000, 4, start)


def test_one_cell_many_times():
    """A list that names a cell for many positions, and the same expert for every pair of a token."""
    n, start, heads, kvh, d = 40, 400, 4, 1, 128
    g = torch.Generator().manual_seed(7)
    k, v = (torch.randn(30, kvh * d, generator=g).half().cuda() for _ in range(2))
    index = (torch.arange(start + n) % 30 // 3).int().cuda()
    chunk(k, v, torch.randn(n, heads * d, generator=g).cuda(), heads, kvh, d, 0.1, 300, 2, start, index)
