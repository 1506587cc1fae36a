"""The router on both sides of the number of scores from which the matrix cores take it,
at rows shorter than a block's step and at long ones, against float64: choices are equal,
a weight is the float64 value rounded once, and a float64 exponential."""

import pytest
import torch

from molla_amd import gpu, synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("experts,tokens", [(7, 4096), (64, 448), (128, 224), (512, 56)])
@pytest.mark.parametrize("width", [4, 36, 256, 4096, 8196])
def test_both_sides(experts, tokens, width):
    ctx, used = gpu.DeviceContext(0), min(experts, 6)
    x = synth.normal((tokens + 3) * width, 1, "cuda").view(-1, width)
    router = synth.normal(experts * width, 2, "cuda", std=2.0 / width ** 0.5).view(experts, width)
    router[experts // 2] = router[1]  # a tie in every row
    logits = x.double() @ router.double().T.contiguous()
    logits[:, experts // 2] = logits[:, 1]
    p = torch.softmax(logits, 1)
    top = torch.sort(p, dim=1, descending=True, stable=True)
    want = top.indices[:, :used]
    w = p.gather(1, want)
    w = w / w.sum(1, keepdim=True)
    for n in (tokens - 1, tokens, tokens + 3):  # 28672 scores from the second on
        ids = torch.full((n, used), -5, dtype=torch.int32, device="cuda")
        weights = torch.zeros(n, used, device="cuda")
        gpu.device_router(ctx, x[:n], router, ids, weights)
        assert torch.equal(ids, want[:n].int())
        assert ((weights.double() - w[:n]).abs() <= 2.0 ** -23 * w[:n]).all()
