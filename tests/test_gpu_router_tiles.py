"""The router over many tokens, at each width of its blocks and at sizes that are no
whole number of them, against float64.  Choices are equal, ties and near scores
included; a weight is the float64 value rounded once, and a float64 exponential."""

import pytest
import torch

from molla_amd import gpu, synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,experts,width", [(4100, 17, 1028), (2050, 60, 1020), (2050, 64, 2048), (4100, 33, 516),
                                                  (2050, 100, 1028), (2050, 128, 1024), (1030, 128, 1052), (1030, 200, 736),
                                                  (300, 512, 1060), (2300, 16, 2052), (140, 512, 1000)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_router(tokens, experts, width, sigmoid):
    used = min(experts, 6)
    x = synth.normal(tokens * width, 1, "cuda").view(tokens, width)
    router = synth.normal(experts * width, 2, "cuda", std=2.0 / width ** 0.5).view(experts, width)
    router[experts // 2] = router[1]  # a tie in every row
    bias = synth.normal(experts, 3, "cuda", std=0.02) if sigmoid else None
    if sigmoid:
        bias[experts // 2] = bias[1]
    ids = torch.full((tokens, used), -5, dtype=torch.int32, device="cuda")
    weights = torch.zeros(tokens, used, device="cuda")
    gpu.device_router(gpu.DeviceContext(0), x, router, ids, weights, bias=bias, sigmoid=sigmoid, norm=not sigmoid)
    logits = x.double() @ router.double().T.contiguous()
    logits[:, experts // 2] = logits[:, 1]
    p = torch.sigmoid(logits) if sigmoid else torch.softmax(logits, 1)
    want = torch.sort(p if bias is None else p + bias.double(), dim=1, descending=True, stable=True).indices[:, :used]
    w = p.gather(1, want)
    if not sigmoid:
        w = w / w.sum(1, keepdim=True)
    assert torch.equal(ids, want.int())
    assert ((weights.double() - w).abs() <= 2.0 ** -23 * w).all()
