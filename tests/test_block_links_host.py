"""What link_records says of a chain of layers, and when it is asked again. No device is touched."""
import numpy as np

from nervanagpu_b200.layers import ConvLayer, FullLayer, link_records


def test_links_follow_the_layers_when_they_change():
    """A chain linked with records and again without: every layer masks its deltas itself then, as the one above keeps no record."""
    below = ConvLayer(None, np.float16, 8, 8, 16, H=4, W=4, R=3, S=3, pad_h=1, pad_w=1)
    above = FullLayer(None, np.float16, 8, 16 * 16, 24, checkpoint=True)
    assert link_records([below, above]) == [True, False]
    assert below.masked_above and above.masks_below
    above.checkpoint = False
    assert link_records([below, above]) == [False, False]
    assert not below.masked_above and not above.masks_below


def test_chains_that_share_a_layer_keep_each_others_links():
    """A chain linked in two parts, the second of which starts with the layer that ends the first."""
    first = ConvLayer(None, np.float16, 8, 8, 16, H=4, W=4, R=3, S=3, pad_h=1, pad_w=1)
    middle = ConvLayer(None, np.float16, 8, 16, 16, H=4, W=4, R=3, S=3, pad_h=1, pad_w=1, checkpoint=True)
    last = FullLayer(None, np.float16, 8, 16 * 16, 24, checkpoint=True)
    assert link_records([first, middle]) == [True, False] and link_records([middle, last]) == [True, False]
    assert first.masked_above and middle.masks_below and middle.masked_above and last.masks_below
