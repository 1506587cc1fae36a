"""The decoder layer over trees of drafted tokens with the weights of a Q4_K_M file
(Q6_K values and down projections): its q and k leave the matvecs unrotated, in the
launches that rotate and store for a plain step."""

import pytest
import torch

import oracle
from molla_amd import block, gpu
from tests.test_gpu_layer import device_layer_from, make_layer_weights, spec_of
from tests.test_gpu_tree_layer import Trees, run

pytestmark = pytest.mark.gpu

KINDS = {"wv": oracle.Q6_K, "down": oracle.Q6_K}


@pytest.mark.parametrize("form", ["f16", "q8"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("lens,counts", [([33], [1]), ([20], [2]), ([15, 0, 40], [1, 1, 1]), ([15, 0, 40], [3, 4, 1]),
                                         ([20, 0, 40], [13, 5, 0])])
def test_mixed_layer(form, paged, lens, counts):
    spec = spec_of(1024, 2048, 8, 2, 128)
    host = make_layer_weights(spec, 23, KINDS)
    _, layer = device_layer_from(host, spec)
    run(spec, host, layer, lens, counts, form, paged)


@pytest.mark.parametrize("neox", [0, 1])
@pytest.mark.parametrize("counts", [[1], [2, 1], [5, 3]])
def test_mixed_layer_pairings(neox, counts):
    spec = dict(spec_of(1024, 2048, 8, 2, 128), neox=neox)
    host = make_layer_weights(spec, 24, KINDS)
    _, layer = device_layer_from(host, spec)
    run(spec, host, layer, [30, 7][:len(counts)], counts, "f16", True)


@pytest.mark.parametrize("counts", [[1, 1], [4, 4]])
def test_chained_mixed_layers(counts):
    spec = spec_of(1024, 2048, 8, 2, 128)
    outs = []
    for chained in (False, True):
        ctx = gpu.DeviceContext(0)
        layers = [device_layer_from(make_layer_weights(spec, 70 + i, KINDS), spec)[1] for i in range(3)]
        if chained:
            block.chain_layers([layer.desc for layer in layers])
        s = Trees(ctx, spec, [12, 30], counts, "f16", True, layers=3)
        s.plan()
        for i, layer in enumerate(layers):
            s.layer(layer, i)
        ctx.synchronize()
        outs.append([s.xd] + s.k + s.v)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_layer_of_many_sequences():
    """More sequences than a wave has lanes, a token each, some without one."""
    spec = spec_of(512, 1024, 8, 2, 64)
    host = make_layer_weights(spec, 25)
    _, layer = device_layer_from(host, spec)
    run(spec, host, layer, [(7 * i) % 40 for i in range(70)], [int(i % 9 != 4) for i in range(70)], "f16", True)
