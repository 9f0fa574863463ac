"""Device memory of networks with 8-bit records, as the benchmark driver lays them out (B200 only)."""
import pytest

from nervanagpu_b200 import NervanaGPU
from nervanagpu_b200 import convnet_benchmarks as cb
from nervanagpu_b200.layers import DataLayer

pytestmark = pytest.mark.gpu


def activation_bytes(layers):
    """Of outputs, records and restored inputs, each buffer once (its largest user counts)."""
    buffers = {}
    for layer in layers:
        if isinstance(layer, DataLayer):
            continue
        own = [layer.fprop_out, getattr(layer, "restored", None)]
        if layer.record is not None:
            own += [layer.record.codes, layer.record.scales]
        for t in own:
            if t is not None:
                buffers[t.ptr] = max(buffers.get(t.ptr, 0), t.nbytes)
    return sum(buffers.values())


def test_a_chain_of_equal_layers_takes_two_outputs_and_its_records():
    """Six convolutions and a fully-connected layer: without records six outputs of 2 bytes per number; with them six
    records (the first convolution's input is data and has none) of 36 bytes per row of 32 images, and two outputs in turn,
    one of which holds what is restored in the backward pass."""
    ng = NervanaGPU(stochastic_round=False)
    confs = [cb._data(32, 16, 12)] + [cb._conv(16, 3, pad=1)] * 6 + [cb._full(8)]
    unit = 16 * 12 * 12 * 32
    plain = activation_bytes(cb.build_network(ng, confs))
    kept = activation_bytes(cb.build_network(ng, confs, checkpoint=True))
    last = 8 * 32 * 2
    assert plain == 6 * 2 * unit + last
    assert kept == 2 * 2 * unit + 6 * unit * 36 // 32 + last


def test_the_two_buffers_are_as_large_as_their_own_layers_need():
    ng = NervanaGPU(stochastic_round=False)
    confs = [cb._data(32, 16, 12), cb._conv(64, 3, pad=1), cb._conv(16, 3, pad=1), cb._conv(32, 3, pad=1), cb._conv(8, 3, pad=1), cb._full(8)]
    layers = cb.build_network(ng, confs, checkpoint=True)
    map_ = 12 * 12 * 32
    assert activation_bytes(layers) == 2 * map_ * (64 + 16) + map_ * (64 + 16 + 32 + 8) * 36 // 32 + 8 * 32 * 2
    assert layers[1].fprop_out.ptr == layers[3].fprop_out.ptr != layers[2].fprop_out.ptr == layers[4].fprop_out.ptr
