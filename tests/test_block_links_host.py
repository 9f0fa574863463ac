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
    above.checkpoint = True
    link_records([below, above])
    assert link_records([above]) == [False] and not above.masks_below
