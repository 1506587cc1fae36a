"""The experts' MLP gives the same bits each time, on every way that it may take: the
slots that atomics number and the order of the weighted sum go into none of them."""

import pytest
import torch

from molla_amd import gpu, synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kinds", [(gpu.Q_Q4_K, gpu.Q_Q4_K), (gpu.Q_Q4_K, gpu.Q_Q6_K), (gpu.Q_Q8_0, gpu.Q_Q8_0)])
@pytest.mark.parametrize("experts,tokens,used", [(8, 1, 3), (6, 2, 2), (4, 8, 2), (4, 6, 4), (8, 40, 2), (5, 333, 3)])
def test_repeated(kinds, experts, tokens, used):
    width, hidden = 512, 768
    w = [gpu.Tensor.from_bytes(synth.quant_tensor(k, experts * r, c, i, device="cuda"), k, c, experts * r)
         for i, (k, r, c) in enumerate(((kinds[0], hidden, width), (kinds[0], hidden, width), (kinds[1], width, hidden)))]
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, width, generator=g).cuda()
    ids = torch.stack([torch.randperm(experts, generator=g)[:used] for _ in range(tokens)]).int()
    ids[::3, 0] = 1
    ids[0, -1] = ids[0, 0]  # one expert twice
    if tokens > 4:
        ids[4, 0] = -1
    ids = ids.cuda()
    weights = torch.rand(tokens, used, generator=g).cuda()
    outs = []
    for i in range(6):
        out = torch.full((tokens, width), float(i), device="cuda")
        gpu.device_experts_mlp(gpu.DeviceContext(0), *w, experts, x, ids, weights, out)
        outs.append(out)
    assert torch.isfinite(outs[0]).all()
    assert all(torch.equal(outs[0], o) for o in outs[1:])
