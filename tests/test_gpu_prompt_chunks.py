"""Prompts whose last chunk wants a larger workspace than a whole one (its products are
cut into more parts)."""

import ctypes

import pytest
import torch

from molla_amd import _lib, block, gpu, synth

pytestmark = pytest.mark.gpu


def test_a_shorter_last_chunk():
    spec = block.BlockSpec(width=1024, hidden=4096, heads=8, kv_heads=2, head_dim=128, rope_dim=128)
    shapes = dict(wq=(1024, 1024), wk=(256, 1024), wv=(256, 1024), wo=(1024, 1024), gate=(4096, 1024), up=(4096, 1024),
                  down=(1024, 4096))
    weights = {n: gpu.Tensor.from_bytes(synth.quant_tensor(gpu.Q_Q4_K, r, c, i), gpu.Q_Q4_K, c, r)
               for i, (n, (r, c)) in enumerate(shapes.items())}
    norm = lambda s: synth.normal(1024, s, "cuda", mean=1.0, std=0.1)
    steps = torch.from_numpy(gpu.rope_steps(128, spec.rope_base)).cuda()
    layer = block.DeviceLayer(spec, norm(20), norm(21), weights, steps)
    size = lambda n: _lib.lib().mi_layer_workspace(ctypes.byref(layer.desc), 600, n)
    assert size(256) > size(257)
    head = gpu.Tensor.from_bytes(synth.quant_tensor(gpu.Q_Q6_K, 512, 1024, 9), gpu.Q_Q6_K, 1024, 512)
    model = block.DeviceModel(spec, synth.normal(512 * 1024, 5, "cuda").view(512, 1024), [layer], norm(6), head)
    ids = synth.tokens(513, 512, 3).cuda()
    rows = []
    for chunk in (257, 171):
        ses = block.DeviceSession(gpu.DeviceContext(0), model, 1, 600)
        ses.prefill(ids, 0, chunk=chunk)
        torch.cuda.synchronize()
        rows.append(ses.x.clone())
    # (the two cut the same sums differently: float32 rounding of a layer's outputs)
    assert (rows[0] - rows[1]).abs().max() <= 1e-4 * rows[0].abs().max()
