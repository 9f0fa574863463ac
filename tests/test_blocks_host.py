"""Matrices in blocks: what is refused, sizes, views and the oracle's definition. No device is touched."""
import ctypes

import numpy as np
import pytest

from nervanagpu_b200 import NervanaGPU, _lib
from nervanagpu_b200.blocks import FORMATS, BlockTensor
from oracle import reference_math as rm


class Host(NervanaGPU):
    """A backend whose launches would fail: everything here has to be refused before."""

    def __init__(self):
        self.lib, self.stream, self.bench, self.round_mode, self.rand_state = _lib.load(), None, False, 0, None


def block(ng, shape, fmt, axis=1, scale=1.0, address=1 << 20):
    desc = _lib.BlockDesc(FORMATS[fmt], axis, shape[0], shape[1], 0, scale, address, address + (1 << 24))
    return BlockTensor(ng, shape, fmt, axis, scale, desc=desc)


def test_shapes_axes_and_scales_that_are_refused():
    ng = Host()
    for shape, fmt, axis, scale, error in [((4, 4), "int8", 1, 1.0, ValueError), ((4,), "mxfp4", 1, 1.0, AssertionError),
                                           ((4, 4, 4), "mxfp4", 1, 1.0, AssertionError), ((4, 4), "mxfp4", 2, 1.0, AssertionError),
                                           ((0, 4), "mxfp8", 1, 1.0, AssertionError), ((4, 0), "mxfp8", 1, 1.0, AssertionError),
                                           ((4, 4), "mxfp8", 1, 2.0, AssertionError), ((4, 4), "nvfp4", 1, 3.0, AssertionError),
                                           ((4, 4), "nvfp4", 1, 0.0, AssertionError), ((4, 4), "nvfp4", 1, float("nan"), AssertionError),
                                           ((4, 4), "nvfp4", 1, -2.0, AssertionError), ((4, 4), "nvfp4", 1, float("inf"), AssertionError)]:
        with pytest.raises(error):
            ng.block_empty(shape, fmt, axis=axis, scale=scale)


def test_operands_that_are_refused(fake_tensor):
    ng = Host()
    X, Q4, Q8 = fake_tensor((64, 32)), block(ng, (64, 32), "nvfp4", 0), block(ng, (64, 32), "mxfp8")
    with pytest.raises(AssertionError):
        ng.quantize(X)
    with pytest.raises(AssertionError):
        ng.quantize(X, Q4, Q4, Q4, Q4, Q4)
    with pytest.raises(AssertionError):
        ng.quantize(X, X)
    with pytest.raises(AssertionError):
        ng.quantize(fake_tensor((32, 64)), Q4)
    with pytest.raises(TypeError):
        ng.quantize(fake_tensor((64, 32), np.int32), Q4)
    with pytest.raises(TypeError):
        ng.dequantize(Q4, fake_tensor((64, 32), np.uint8))
    with pytest.raises(TypeError):
        ng.relu_mask(Q4, X)
    with pytest.raises(AssertionError):
        ng.relu_mask(Q8, fake_tensor((64, 33)))
    W, C = block(ng, (16, 64), "nvfp4"), fake_tensor((16, 32))
    for a, b, c, error in [(W, X, C, AssertionError), (W, block(ng, (64, 32), "mxfp4", 0), C, TypeError), (W, Q8, C, TypeError),
                           (W, block(ng, (64, 32), "nvfp4", 1), C, AssertionError), (W.T.T.T, Q4, C, AssertionError),
                           (block(ng, (16, 64), "nvfp4", 0), Q4, C, AssertionError), (W, block(ng, (65, 32), "nvfp4", 0), C, AssertionError),
                           (W, Q4, fake_tensor((32, 16)).T, AssertionError), (W, Q4, fake_tensor((16, 32), np.int32), TypeError),
                           (W, Q4, fake_tensor((16, 33)), AssertionError), (W, Q4, fake_tensor((16, 64))[:, ::2], AssertionError),
                           (W, Q4, fake_tensor((16, 32))[::-1], AssertionError),
                           (block(ng, (16, 64), "mxfp8"), block(ng, (64, 32), "mxfp8", 0), C, TypeError),
                           (fake_tensor((16, 64)), Q4, C, TypeError), (fake_tensor((16, 64), np.float32), Q8, C, TypeError),
                           (fake_tensor((16, 64)), Q8, C, AssertionError), (fake_tensor((64, 16)).T, block(ng, (64, 32), "mxfp8", 0), C, AssertionError)]:
        with pytest.raises(error):
            ng.block_dot(a, b, c)


def test_c_entries_refuse_before_they_touch_a_device(lib):
    D, byref, null = _lib.BlockDesc, ctypes.byref, None
    good4 = D(1, 1, 16, 64, 0, 1.0, 1 << 20, 1 << 21)
    other = D(1, 0, 64, 32, 0, 1.0, 1 << 20, 1 << 21)
    good8 = D(2, 0, 64, 32, 0, 1.0, 1 << 20, 1 << 21)
    a, b = ctypes.c_size_t(), ctypes.c_size_t()

    def bad(rc, code=-1):
        assert rc == code, (rc, lib.ng_last_error())

    for fields, code in [((3, 1, 4, 4), -1), ((-1, 1, 4, 4), -1), ((0, 2, 4, 4), -1), ((0, 1, 0, 4), -1), ((0, 1, 4, -1), -1),
                         ((0, 1, 2 ** 31 - 1, 4), -8)]:
        d = D(*fields, 0, 1.0, 1 << 20, 1 << 21)
        bad(lib.ng_block_bytes(byref(d), byref(a), byref(b)), code)
        bad(lib.ng_block_quantize(1 << 20, 2, 1, 1, byref(d), 1, null), code)
        bad(lib.ng_block_dequantize(byref(d), 1 << 20, 2, 1, 1, null), code)
        bad(lib.ng_block_relu_mask(byref(d), 1 << 20, 2, 1, 1, null), code)
        bad(lib.ng_block_dot(byref(d), byref(other), 1 << 20, 32, 0, 1, 0, 0, 0, 0, 0, null), code)
        bad(lib.ng_block_dot_f16(1 << 20, 64, byref(d), 1 << 20, 16, 32, 0, 1, 0, 0, 0, 0, 0, null), code)
    for scale in (0.0, -1.0, 3.0, float("nan"), float("inf"), 2.0 ** 33, 2.0 ** -33):
        bad(lib.ng_block_bytes(byref(D(1, 1, 4, 4, 0, scale, null, null)), byref(a), byref(b)))
    bad(lib.ng_block_bytes(byref(D(0, 1, 4, 4, 0, 2.0, null, null)), byref(a), byref(b)))
    bad(lib.ng_block_bytes(null, byref(a), byref(b)))
    bad(lib.ng_block_bytes(byref(good4), null, byref(b)))
    bad(lib.ng_block_quantize(null, 2, 1, 1, byref(good4), 1, null))
    bad(lib.ng_block_quantize(1 << 20, 8, 1, 1, byref(good4), 1, null), -2)
    bad(lib.ng_block_quantize(1 << 20, 2, 1, 1, byref(good4), 0, null))
    bad(lib.ng_block_quantize(1 << 20, 2, 1, 1, byref(good4), 5, null))
    bad(lib.ng_block_quantize(1 << 20, 2, 1, 1, (D * 2)(good4, other), 2, null))
    bad(lib.ng_block_relu_mask(byref(good4), 1 << 20, 2, 1, 1, null), -2)
    bad(lib.ng_block_dot(byref(good4), byref(good4), 1 << 20, 64, 0, 1, 0, 0, 0, 0, 0, null), -2)      # axes
    bad(lib.ng_block_dot(byref(good4), byref(good8), 1 << 20, 64, 0, 1, 0, 0, 0, 0, 0, null), -2)      # formats
    bad(lib.ng_block_dot(byref(good4), byref(other), 1 << 20, 31, 0, 1, 0, 0, 0, 0, 0, null))          # ldc
    bad(lib.ng_block_dot(byref(good4), byref(other), null, 32, 0, 1, 0, 0, 0, 0, 0, null))
    bad(lib.ng_block_dot(byref(good4), byref(other), 1 << 20, 32, 0, 1, 0, 0, 11, 0, 0, null))
    bad(lib.ng_block_dot(byref(good4), byref(other), 1 << 20, 32, 1, 1, 0, 0, 10, 0, 0, null), -2)     # stochastic fp32
    bad(lib.ng_block_dot_f16(1 << 20, 63, byref(good8), 1 << 20, 16, 32, 0, 1, 0, 0, 0, 0, 0, null))   # lda
    bad(lib.ng_block_dot_f16(1 << 20, 64, byref(good8), 1 << 20, 0, 32, 0, 1, 0, 0, 0, 0, 0, null))
    bad(lib.ng_block_dot_f16(1 << 20, 64, byref(other), 1 << 20, 16, 32, 0, 1, 0, 0, 0, 0, 0, null), -2)


@pytest.mark.parametrize("fmt,axis,shape,codes,scales", [
    ("mxfp4", 1, (1, 1), 2048, 1024), ("nvfp4", 1, (1, 1), 2048, 2048), ("mxfp8", 1, (1, 1), 32, 4), ("mxfp8", 1, (100, 64), 6400, 400), ("mxfp8", 1, (100, 129), 16000, 800),
    ("nvfp4", 1, (20, 257), 32 * 256, 4096), ("mxfp4", 1, (64, 256), 64 * 128, 1024), ("mxfp4", 1, (65, 256), 128 * 128, 1024),
    ("nvfp4", 1, (129, 257), 256 * 256, 2 * 4096), ("mxfp4", 0, (257, 129), 256 * 256, 2 * 2048), ("mxfp8", 0, (257, 129), 129 * 288, 129 * 12),
    ("nvfp4", 1, (70000, 70000), 547 * 274 * 16384, 547 * 274 * 2048)])
def test_sizes(lib, fmt, axis, shape, codes, scales):
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    d = _lib.BlockDesc(FORMATS[fmt], axis, shape[0], shape[1], 0, 1.0, None, None)
    assert lib.ng_block_bytes(ctypes.byref(d), ctypes.byref(a), ctypes.byref(b)) == 0
    assert (a.value, b.value) == (codes, scales)


def test_transposed_views_share_memory():
    ng = Host()
    q = block(ng, (16, 64), "nvfp4", 1, 2.0 ** -4)
    t = q.T
    assert t.shape == (64, 16) and t.axis == 0 and t.scale == q.scale and t.desc.codes == q.desc.codes
    assert (t.desc.rows, t.desc.cols, t.desc.axis) == (64, 16, 0) and t.T.shape == q.shape and t.T.axis == 1
    assert "nvfp4" in str(q) and q.size == 1024


def test_a_transposed_view_is_made_once_and_holds_no_cycle():
    import weakref
    q = block(Host(), (16, 64), "mxfp8", 1, 1.0)
    t, gone = q.T, weakref.ref(q)
    assert q.T is t
    del q
    assert gone() is None and t.shape == (64, 16)       # (freed at once, not by the collector)


def test_block_descriptor_matches_header():
    assert [f[0] for f in _lib.BlockDesc._fields_] == "format axis rows cols device scale codes scales".split()
    assert ctypes.sizeof(_lib.BlockDesc) == 40


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_oracle_rounds_to_the_nearest_of_the_formats_numbers(fmt):
    """The definition itself: errors of at most half a step, exact powers, unchanged by a second pass."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((20, 160)) * np.exp(2 * rng.standard_normal((20, 1)))
    v = rm.block_values(x, fmt)
    block, top = rm.BLOCK_FORMATS[fmt]
    amax = np.repeat(np.abs(x).reshape(20, -1, block).max(axis=2), block, axis=1)
    # E4M3: half of 2^-3 of the value, or of 2^-9 of a scale <= 2 max / 448 (a whole such step where zero is ruled out)
    # E2M1: half of the largest step 2 / 6 of max, after a scale that may be a factor of two up, or E4M3-rounded down
    tol = np.maximum(np.abs(x) / 16, amax / 224 * 2.0 ** -9) if fmt == "mxfp8" else amax * (2.0 / 6 if fmt == "mxfp4" else 0.5 / 3 * 1.0625 + 1.0 / 16)
    assert (np.abs(v - x) <= tol).all()
    assert np.array_equal(rm.block_values(v, fmt), v) or fmt == "nvfp4"
    if fmt == "mxfp8":
        assert np.array_equal(v > 0, x > 0)
