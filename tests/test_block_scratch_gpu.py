"""Products of an 8-bit record that may use scratch memory, when there is some of it or none (B200 only)."""
import ctypes

import numpy as np
import pytest

from nervanagpu_b200 import NervanaGPU
from oracle import reference_math as rm
from tests._util import assert_close
from tests.test_blocks_gpu import product_tol

pytestmark = pytest.mark.gpu


def fallbacks(ng):
    n = ctypes.c_ulonglong()
    assert ng.lib.ng_fallback_launch_count(ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("odd", [0, 1])
def test_a_recording_with_room_for_the_copy_and_none_for_the_product(odd):
    """4096 x 4096 x 2048, a sum in one part, makes room for a copy of the record on a new stream and for nothing else. 600 x 500 x
    8200 on that stream would take a copy, which fits, and then parts of its sum (and A's odd rows put in order), which do
    not: a recording of it takes the form without scratch memory, on the tensor cores."""
    ng = NervanaGPU(stochastic_round=False)
    rng = np.random.default_rng(odd)
    ng.stream = ng.new_stream()
    big = ng.quantize(ng.ones((4096, 2048)), ng.block_empty((4096, 2048), "mxfp8"))
    ng.block_dot(ng.ones((4096, 2048)), big.T, ng.empty((4096, 4096)))
    m, n, k = 600, 500, 8200
    E = np.full((m, k + odd), np.nan, np.float16)
    E[:, odd:] = rng.standard_normal((m, k)) * 0.1
    X = np.maximum(rng.standard_normal((n, k)), 0).astype(np.float16)
    A, Q = ng.array(E)[:, odd:], ng.quantize(ng.array(X), ng.block_empty((n, k), "mxfp8"))
    C = ng.zeros((m, n), dtype=np.float32)
    ng.synchronize()
    x, e = rm.block_values(X, "mxfp8"), E[:, odd:].astype(np.float64)
    ref, mag = e @ x.T, np.abs(e) @ x.T
    before = fallbacks(ng)
    run = ng.capture(lambda: ng.block_dot(A, Q.T, C))
    run.launch()
    assert_close(C.get(), ref, product_tol(ref, mag, k, f32=True))
    ng.block_dot(A, Q.T, C)                 # (and live, with room)
    assert_close(C.get(), ref, product_tol(ref, mag, k, f32=True))
    assert fallbacks(ng) == before
