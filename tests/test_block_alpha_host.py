"""Factors of a 4-bit product that fp32 cannot hold together with the operands' scales are refused. No device is touched."""
import ctypes

import pytest

from nervanagpu_b200 import _lib


@pytest.mark.parametrize("alpha,scale", [(1e-30, 2.0 ** -32), (1e30, 2.0 ** 32), (-1e30, 2.0 ** 32), (1.2345678 * 2.0 ** -126, 0.5)])
def test_a_factor_beyond_fp32_is_refused(lib, alpha, scale):
    D, byref = _lib.BlockDesc, ctypes.byref
    A, B = (D(1, axis, *shape, 0, scale, 1 << 20, 1 << 21) for axis, shape in ((1, (16, 64)), (0, (64, 32))))
    rc = lib.ng_block_dot(byref(A), byref(B), 1 << 20, 32, 1, alpha, 0, 0, 0, 0, 0, None)
    assert rc == -2 and b"alpha" in lib.ng_last_error()
