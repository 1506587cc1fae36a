"""The decoder layer with experts whose width is no multiple of 256, against the float64
layer of test_gpu_sparse_layer.py."""

import pytest

from molla_amd import gpu
from tests.test_gpu_sparse_layer import Layer, Run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden,kinds", [
    (64, (gpu.Q_Q4_K, gpu.Q_Q4_K, gpu.Q_Q8_0)), (192, (gpu.Q_Q8_0,) * 3), (320, (gpu.Q_Q4_K, gpu.Q_Q6_K, gpu.Q_Q4_0)),
    (1408, (gpu.Q_Q4_K, gpu.Q_Q4_K, gpu.Q_Q5_0))])
@pytest.mark.parametrize("lens,chunk", [((44,), 0), ((44, 5, 19, 30, 8), 0), ((40,), 20), ((3,), 90)])
def test_widths(hidden, kinds, lens, chunk):
    r = Run(Layer(hidden=hidden, kinds=kinds), lens, "f16", False, chunk)
    # (of a chunk the rows of the other layer tests.  These layers' scores are of about
    # 1000, sums of products of 4000: off by 4000 * 2^-20 = 0.004.  Where a head's two
    # largest lie within 1 of each other, as in row 73 of 90 two heads' do, that moves
    # their weights by 1e-3 and the row by more than the gate's 1e-4, whatever the
    # experts' width)
    r.check(r.go(gpu.DeviceContext(0)), rows=sorted({0, 1, chunk // 2, chunk - 1}) if chunk else None)
