"""block.DeviceLayer looks at the router that it passes on by its address: as many
values as the experts have, one after another (on the host, with weights made up)."""

import pytest
import torch

from molla_amd import _lib, block

SPEC = dict(width=256, heads=4, kv_heads=2, head_dim=64, rope_dim=64, rope_base=10000.0, hidden=512)


class Weight:
    def weight(self):
        return _lib.MiWeight()


class Device(torch.Tensor):
    """A host tensor in the place of one on the device."""
    is_cuda = True


def layer(router=None, bias=None, experts=6):
    extras = {n: t.as_subclass(Device) for n, t in (("router", router), ("router_bias", bias)) if t is not None}
    w = torch.ones(256)
    return block.DeviceLayer(block.BlockSpec(**SPEC, experts=experts, experts_used=2), w, w,
                             {n: Weight() for n in block.DeviceLayer.NAMES}, torch.ones(32), extras=extras)


@pytest.mark.parametrize("router,bias", [
    (torch.ones(6 * 256), None), (torch.ones(6, 256), torch.ones(6)), (torch.ones(6, 256), None)])
def test_taken(router, bias):
    d = layer(router, bias).desc
    assert d.router == router.data_ptr() and (d.router_bias or 0) == (0 if bias is None else bias.data_ptr())


@pytest.mark.parametrize("router,bias,words", [
    (None, None, "router"), (torch.ones(3 * 256), None, "router"), (torch.ones(6, 255), None, "router"),
    (torch.ones(7, 256), None, "router"), (torch.ones(256, 6).t(), None, "router"), (torch.ones(256, 6), None, "router"), (torch.ones(6, 512)[:, :256], None, "router"),
    (torch.ones(6, 256), torch.ones(5), "router_bias"), (torch.ones(6, 256), torch.ones(256), "router_bias"),
    (torch.ones(6, 256), torch.ones(12)[::2], "router_bias"), (torch.ones(6, 256).half(), None, "float32")])
def test_refused(router, bias, words):
    with pytest.raises(ValueError, match=words):
        layer(router, bias)



def test_a_layer_without_experts_needs_none():
    layer(experts=0)
    layer(torch.ones(6, 256), experts=0)  # (nor reads one)
