"""Scratch memory that the device does not have (B200 only)."""
import ctypes

import numpy as np
import pytest

from nervanagpu_b200 import NervanaGPU

pytestmark = pytest.mark.gpu


def test_memory_that_is_refused_again_and_again_is_not_lost():
    """A copy of 2.7 GB with 1.5 GB left: the product runs without it. Beside a living recording, and with other calls that use
    the same scratch buffer in between, this neither loses what the buffer was nor takes more memory each time."""
    ng = NervanaGPU(stochastic_round=False)
    ng.stream = ng.new_stream()
    lib = ng.lib

    def free_bytes():
        free, total = ctypes.c_size_t(), ctypes.c_size_t()
        assert lib.ng_mem_info(ctypes.byref(free), ctypes.byref(total)) == 0
        return free.value

    n, k, m = 16384, 65536, 128
    X = ng.empty((n, k))
    X.fill(1)
    Q = ng.quantize(X, ng.block_empty((n, k), "mxfp8"))
    del X
    A, C = ng.ones((m, k + 1))[:, 1:], ng.empty((m, n), dtype=np.float32)      # (odd rows: the copy is the rule's choice)
    small = ng.quantize(ng.ones((4096, 2048)), ng.block_empty((4096, 2048), "mxfp8"))      # a copy of 16 MB, in the same buffer
    E, D = ng.ones((4096, 2048)), ng.empty((4096, 4096))
    ng.block_dot(E, small.T, D)
    keep = ng.capture(lambda: ng.block_dot(E, small.T, D))
    ng.synchronize()
    room = ctypes.c_void_p()
    assert lib.ng_malloc(ctypes.byref(room), free_bytes() - (3 << 29)) == 0
    try:
        free = []
        for _ in range(4):
            C.fill(0)
            ng.block_dot(A, Q.T, C)
            assert (C.get() == k).all()
            D.fill(0)
            ng.block_dot(E, small.T, D)
            assert (D.get() == 2048).all()
            free.append(free_bytes())
        assert min(free) == max(free), free
    finally:
        assert lib.ng_free(room) == 0
    ng.block_dot(A, Q.T, C)                 # with memory again
    assert (C.get() == k).all()
    keep.launch()
    assert (D.get() == 2048).all()
    keep.release()
