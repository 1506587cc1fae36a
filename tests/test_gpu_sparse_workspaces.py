"""Calls of every size on the workspace of the largest, among bytes that stay as they
were: fewer tokens take other kernels, cut into more parts."""

import pytest
import torch

from molla_amd import gpu, synth

pytestmark = pytest.mark.gpu


def room(need):
    held = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
    return held, held[256:256 + need]


def kept(held):
    torch.cuda.synchronize()
    assert (held[:256] == 77).all() and (held[-256:] == 77).all()


@pytest.mark.parametrize("kinds", [(gpu.Q_Q4_K, gpu.Q_Q4_K), (gpu.Q_Q4_K, gpu.Q_Q6_K), (gpu.Q_Q8_0, gpu.Q_Q8_0)])
@pytest.mark.parametrize("most", [5, 21, 40, 130])
@pytest.mark.parametrize("width,hidden", [(256, 4352), (1024, 512)])
def test_experts(kinds, most, width, hidden):
    experts, used = 8, 4
    c, L = gpu.DeviceContext(0), gpu.lib()
    mk = lambda k, r, n, s: gpu.Tensor.from_bytes(synth.quant_tensor(k, experts * r, n, s), k, n, experts * r)
    gate, up, down = mk(kinds[0], hidden, width, 1), mk(kinds[0], hidden, width, 2), mk(kinds[1], width, hidden, 3)
    d = gpu.MiExperts(experts, width, hidden, 0, gate.weight(), up.weight(), down.weight())
    held, work = room(L.mi_experts_workspace(d, most, used))
    x = synth.normal(most * width, 6, "cuda", std=0.05).view(most, width)
    g = torch.Generator().manual_seed(most)
    ids = torch.stack([torch.randperm(experts, generator=g)[:used] for _ in range(most)]).int().cuda()
    weights = torch.rand(most, used, generator=g).cuda()
    for n in sorted({1, 2, 3, 5, 8, 13, 16, 17, 20, 33, most - 1, most}):
        if n > most:
            continue
        a, b = torch.zeros(n, width, device="cuda"), torch.zeros(n, width, device="cuda")
        args = experts, x[:n], ids[:n], weights[:n]
        gpu.device_experts_mlp(c, gate, up, down, *args, a, work=work)
        gpu.device_experts_mlp(c, gate, up, down, *args, b)
        assert torch.equal(a, b) and a.abs().max() > 0
    kept(held)


@pytest.mark.parametrize("heads,kvh,d", [(32, 8, 128), (8, 2, 64), (4, 2, 256), (8, 2, 96)])
@pytest.mark.parametrize("form", [gpu.CACHE_F16, gpu.CACHE_Q8])
@pytest.mark.parametrize("most", [9, 40, 300])
@pytest.mark.parametrize("chunk", [False, True])
def test_window(heads, kvh, d, form, most, chunk):
    window, first, positions = 700, 4, 2100
    c, L = gpu.DeviceContext(0), gpu.lib()
    held, work = room(L.mi_attend_window_workspace(heads, kvh, d, form, window, first, positions, most, int(chunk)))
    row = gpu.cache_row(form, kvh * d)
    g = torch.Generator(device="cuda").manual_seed(3)
    # (as q8_0, bytes and half factors: below 0x3c00, so that none is an infinity)
    k, v = (torch.randint(0, 0x3c00, (positions, row), generator=g, device="cuda").short().view(torch.float16)
            for _ in range(2))
    index = None if chunk else torch.arange(positions, device="cuda", dtype=torch.int32).repeat(most, 1)
    q = torch.randn(most, heads * d, generator=g, device="cuda")
    for n in sorted({1, 3, 7, 8, 9, 17, 32, 33, 256, most - 1, most}):
        for count in (2100, 1500, 65):
            if n > most or n > count:
                continue
            pos = torch.arange(count - n, count, dtype=torch.int32, device="cuda")
            a, b = torch.zeros(n, heads * d, device="cuda"), torch.zeros(n, heads * d, device="cuda")
            args = q[:n], k, v, heads, kvh, d, 0.05, window, first, pos, count
            at = None if chunk else index[:n]
            gpu.device_attend_window(c, *args, a, kv_index=at, form=form, work=work)
            gpu.device_attend_window(c, *args, b, kv_index=at, form=form)
            assert torch.equal(a, b) and a.abs().max() > 0
    kept(held)
