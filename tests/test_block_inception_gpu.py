"""Convolutions with 8-bit records inside an Inception's branches (B200 only)."""
import numpy as np
import pytest

from nervanagpu_b200 import NervanaGPU
from nervanagpu_b200 import convnet_benchmarks as cb
from nervanagpu_b200.layers import DataLayer, Inception, Layer
from oracle import reference_math as rm
from tests._util import assert_close, f32_tol

pytestmark = pytest.mark.gpu
f32 = np.float32


def test_records_in_every_layer_of_the_branches():
    ng = NervanaGPU(stochastic_round=False)
    data = DataLayer(ng, np.float16, 32, 16, H=6, W=6)
    record = lambda conf: dict(conf, checkpoint=True)
    conf = {"layer": Inception, "partitions": [[record(cb._conv(8, 1))], [record(cb._conv(16, 1)), record(cb._conv(24, 3, pad=1))]]}
    layer = Layer.create(ng, conf, data, np.float16)
    convs = [l for part in layer.partitions for l in part]
    rng = np.random.RandomState(3)
    data.init_activations()
    data.init_data(np.maximum(rng.standard_normal(data.dimO), 0).astype(np.float16))
    layer.init_activations()
    layer.init_deltas()
    layer.init_weights(rng=rng)
    layer.fprop(data.fprop(None))
    inputs = {l: l.fprop_in.get() for l in convs}
    acts = {l: l.fprop_out.get() for l in convs}
    E = (rng.uniform(-1, 1, layer.dimO) * 0.25).astype(np.float16)
    dE = ng.array(E)
    layer.bprop(dE)
    k0 = 0
    for part in layer.partitions:
        last = part[-1]
        e = np.where(acts[last] > 0, E[k0:k0 + last.K], 0)
        k0 += last.K
        for l in part:
            x = ng.dequantize(l.record, ng.empty(l.dimI2)).get()
            assert np.array_equal(x, rm.block_values(inputs[l].reshape(l.dimI2), "mxfp8").astype(np.float16)) and (x > 0).any()
        C, R = last.C, last.TRS[1]
        cd = rm.ConvDims(32, C, last.K, 1, 6, 6, 1, R, R, 0, last.padding[1], last.padding[2], 1, 1, 1)
        x = x.reshape(last.dimI)
        ref = rm.conv_update_fast(cd, x, e)
        assert_close(last.updat_out.get(), ref, f32_tol(rm.conv_update_fast(cd, np.abs(x.astype(f32)), np.abs(e.astype(f32))), 32 * 36), "dF")
