"""A training step of a whole network with 8-bit records beside the same step without (B200 only)."""
import numpy as np
import pytest

from nervanagpu_b200 import NervanaGPU
from nervanagpu_b200 import convnet_benchmarks as cb
from nervanagpu_b200.layers import ConvLayer, DataLayer, FullLayer, PoolLayer

pytestmark = pytest.mark.gpu


def test_a_step_of_alexnet_with_records_is_that_without_but_for_their_rounding():
    """Both from the same seed. Records change no activation and no mask, so outputs and deltas are equal; a gradient is off by
    what the record's numbers are: an e4m3 number by 2^-4 of the value, or, below its normal range, by 2^-9 of a scale
    of which a block's largest is at least 224 (zero apart, which stays). With E the deltas and X the inputs that is at most 2^-4
    (|E| * |X|) + 2^-9 / 224 (|E| * M), M each block's largest; both products are taken on the device from the plain network's arrays.
    To these come two fp32 sums of t terms, t 2^-23 of (|E| * |X|) each, and (fully-connected layers) two roundings to fp16."""
    ng = NervanaGPU(stochastic_round=False)
    confs = [dict(c, N=32) if c["layer"] is DataLayer else c for c in cb.NETWORKS["Alexnet"][1]]

    def step(checkpoint, seen):
        layers = cb.build_network(ng, confs, seed=7, checkpoint=checkpoint)
        x = None
        for layer in layers:
            x = layer.fprop(x)
        seen(None, x.get(), None, layers)
        rng = np.random.default_rng(1)
        d = ng.array((rng.uniform(-1, 1, layers[-1].dimO) * 0.5).astype(np.float16))
        for layer in layers[:0:-1]:
            e = d
            d = layer.bprop(d)
            seen(layer, e.get().reshape(layer.dimO2), layer.updat_out.get() if layer.weights is not None else None, layers)

    plain = []

    def bounds(layer, e, dw, layers):
        bound = None
        if layer is not None and dw is not None:
            x = layer.fprop_in.get().reshape(layer.dimI2)
            pad = -x.shape[1] % 32
            top = np.pad(x, ((0, 0), (0, pad))).reshape(x.shape[0], -1, 32).max(axis=2)
            top = np.repeat(top, 32, axis=1)[:, :x.shape[1]]
            parts = []
            for v in (np.abs(x), top):
                V, E = ng.array(v), ng.array(np.abs(e))
                out = ng.empty(layer.dimF, dtype=np.float32)
                if isinstance(layer, FullLayer):
                    out = ng.empty(layer.dimF)
                    ng.dot(E, V.T, out)
                else:
                    ng.update_conv(layer, V.reshape(layer.dimI), E.reshape(layer.dimO), out)
                parts.append(out.get().astype(np.float32))
            terms = layer.N * (1 if isinstance(layer, FullLayer) else layer.P * layer.Q)
            bound = (2.0 ** -4 + 2 * terms * 2.0 ** -23) * parts[0] + 2.0 ** -9 / 224 * parts[1]
            bound = bound * (1 + 2.0 ** -9) + 1e-6
            if isinstance(layer, FullLayer):
                bound += 2.0 ** -10 * np.abs(dw.astype(np.float32)) + 2.0 ** -24
        plain.append((e, dw, bound))

    step(False, bounds)
    at = iter(plain)
    checked = []

    def compare(layer, e, dw, layers):
        e0, dw0, bound = next(at)
        assert np.array_equal(e, e0), layer
        if dw is None:
            return
        assert np.isfinite(dw).all() and (dw != 0).any(), layer
        err = np.abs(dw.astype(np.float32) - dw0.astype(np.float32))
        if layer.checkpoint:
            assert (err <= bound).all(), (str(layer), float((err - bound).max()))
            checked.append(layer)
        else:
            assert not err.any(), layer

    step(True, compare)
    assert len([l for l in checked if isinstance(l, ConvLayer)]) == 4 and len(checked) == 7
    assert not any(isinstance(l, PoolLayer) for l in checked)
