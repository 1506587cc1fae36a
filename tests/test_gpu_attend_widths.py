"""Attention at head widths that are no whole number of 64 lanes: the fold of the
slices runs in whole waves, whose sums take every lane."""

import math

import pytest
import torch

from molla_amd import gpu
from tests.test_gpu_tree import FORMS, encode, q8_values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [32, 96, 160, 224, 480])
@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("count", [1, 70, 700])
def test_attend_every_width(d, form, count):
    heads, kvh = 4, 2
    g = torch.Generator().manual_seed(d + count)
    k, v = (encode(torch.randn(count, kvh * d, generator=g), form) for _ in range(2))
    q = torch.randn(heads * d, generator=g)
    out = torch.zeros(heads * d, device="cuda")
    gpu.device_attend(gpu.DeviceContext(0), q.cuda(), k.cuda(), v.cuda(), heads, kvh, d, 1 / math.sqrt(d), count, out,
                      form=FORMS[form])
    kk, vv = (x.double() if form == "f16" else torch.from_numpy(q8_values(x, kvh * d)) for x in (k, v))
    kk, vv = (x.view(count, kvh, d).transpose(0, 1) for x in (kk, vv))
    s = q.double().view(kvh, -1, d) @ kk.transpose(1, 2) / math.sqrt(d)
    want = (torch.softmax(s, -1) @ vv).reshape(-1)
    # a score's d sums of 2^-24 of the absolute products, twice over in a weight, and a
    # rounding of 2^-24 for each key
    size = (q.abs().double().view(kvh, -1, d) @ kk.abs().transpose(1, 2)).max().item() / math.sqrt(d)
    bound = 2.0 ** -24 * vv.abs().max().item() * (2 * d * size + count + 64)
    assert (out.cpu().double() - want).abs().max().item() <= bound
