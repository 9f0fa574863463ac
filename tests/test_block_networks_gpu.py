"""Whole networks through the benchmark driver: records and layer classes of the user's own (B200 only)."""
import numpy as np
import pytest

from nervanagpu_b200 import NervanaGPU
from nervanagpu_b200 import convnet_benchmarks as cb
from nervanagpu_b200.layers import ConvLayer

pytestmark = pytest.mark.gpu


def test_layers_with_an_init_activations_of_their_own():
    """A subclass that overrides init_activations without arguments, as it could before there were records."""
    class Conv(ConvLayer):
        def init_activations(self):
            super(Conv, self).init_activations()
            self.own = True

    ng = NervanaGPU(stochastic_round=False)
    confs = [cb._data(32, 8, 6), dict(cb._conv(16, 3, pad=1), layer=Conv), cb._full(24), cb._full(8)]
    for checkpoint in (False, True):
        layers = cb.build_network(ng, confs, checkpoint=checkpoint)
        x = None
        for layer in layers:
            x = layer.fprop(x)
        assert layers[1].own and np.isfinite(x.get()).all() and (x.get() > 0).any()
