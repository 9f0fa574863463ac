"""Matrices in blocks of small floating-point numbers on the device, against their definition in 64 bits (B200 only).

Quantisation is exact arithmetic up to one rounding per number, so its results have to be equal. Products: the
operands' values are exact on both sides; fp32 sums of k terms on the tensor cores, which may truncate, are off by
at most k * 2^-23 of the sum of magnitudes, and rounding to fp16 by half a step, 2^-11 of the value (2^-25 below the
normal range; a whole step, twice these, when stochastic)."""
import numpy as np
import pytest

from nervanagpu_b200 import NervanaGPU, _lib
from oracle import reference_math as rm
from tests._util import assert_close

pytestmark = pytest.mark.gpu

FORMATS = ["mxfp4", "nvfp4", "mxfp8"]


def product_tol(ref, absdot, k, steps=1.0, f32=False):
    tol = k * 2.0 ** -23 * absdot + 1e-30
    return tol if f32 else tol * (1 + 2.0 ** -10) + steps * (2.0 ** -11 * np.abs(ref) * (1 + 2.0 ** -10) + 2.0 ** -25)


def values(rng, shape, dtype=np.float16, spread=1.5):
    """Rows of different sizes, zeros among the numbers, some blocks of zeros only."""
    x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal((shape[0], 1)))
    x[rng.random(shape) < 0.2] = 0.0
    if shape[1] > 40 and shape[0] > 2:
        x[1, :40] = 0.0
    return x.astype(dtype)


def round_trip(ng, x, fmt, axis, scale=1.0, out_dtype=None):
    A, Q = ng.array(x, dtype=x.dtype), ng.block_empty(x.shape, fmt, axis=axis, scale=scale)
    out = ng.empty(x.shape, dtype=out_dtype or x.dtype)
    out.fill(7.0)
    ng.quantize(A, Q)
    return ng.dequantize(Q, out).get()


def filled(ng, x, fmt, axis, scale=1.0):
    return ng.quantize(ng.array(x, dtype=x.dtype), ng.block_empty(x.shape, fmt, axis=axis, scale=scale))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 17), (31, 1), (3, 8), (33, 65), (128, 128), (130, 257), (257, 1000), (515, 48), (1030, 3), (700, 16), (300, 40), (261, 70)])
def test_round_trip_equals_the_definition(ng, fmt, axis, dtype, shape):
    rng = np.random.default_rng(shape[0] * 1000 + shape[1])
    x = values(rng, shape, dtype)
    scale = 2.0 ** -3 if fmt == "nvfp4" else 1.0
    want = rm.block_values(x, fmt, axis, scale)
    got = round_trip(ng, x, fmt, axis, scale, np.float32)
    assert np.array_equal(got.astype(np.float64), want)
    assert np.array_equal(np.signbit(got[want != 0]), np.signbit(x[want != 0]))
    if dtype is np.float16:
        assert np.array_equal(round_trip(ng, x, fmt, axis, scale), want.astype(np.float16))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_borders_and_extremes(ng, fmt, dtype):
    """Numbers on and next to the borders between two codes, largest magnitudes on and next to those where the scale
    changes, the type's smallest and largest numbers, zeros of both signs."""
    block, top = rm.BLOCK_FORMATS[fmt]
    q = rm.block_numbers(fmt)
    border = (q[1:] + q[:-1]) / 2
    eps = np.finfo(dtype).eps
    near = np.concatenate([border, border * (1 + 2 * eps), border * (1 - 2 * eps), q])
    rows = []
    with np.errstate(over="ignore"):
        for s in (1.0, 1.125, 1.875, 2.0 ** -6, 2.0 ** 5):
            for i in range(0, len(near), block - 1):
                part = near[i:i + block - 1]
                rows.append(np.concatenate([[top], part, np.zeros(block - 1 - len(part))]) * s)
        for m in (top, top * (1 + 2 * eps), top * (1 - 2 * eps), top * 1.0625, top * 1.0625 * (1 + 2 * eps)):
            rows.append(np.concatenate([[m], np.linspace(0, m, block - 1)]))
        fi = np.finfo(dtype)
        for m in (float(fi.max), float(fi.tiny), float(fi.smallest_subnormal), 0.0):
            rows.append(np.concatenate([[m], np.linspace(0, m, block - 1)]))
        x = np.array(rows).astype(dtype)
    assert np.isfinite(x).all()
    x = np.concatenate([x, -x, np.where(np.arange(block) % 2, x, -x)]).astype(dtype)
    for axis in (0, 1):
        xa = x if axis == 1 else np.ascontiguousarray(x.T)
        want = rm.block_values(xa, fmt, axis)
        got = round_trip(ng, xa, fmt, axis, out_dtype=np.float32)
        top = float(np.finfo(np.float32).max)   # (which may itself be rounded to 2^128)
        assert np.array_equal(got, np.clip(want, -top, top).astype(np.float32)), (fmt, axis)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("axis", [0, 1])
def test_numbers_next_to_the_largest_read_back_finite(ng, fmt, axis):
    x = np.array([np.linspace(m / 32, m, 32) * (-1) ** np.arange(32) for m in (65504, 63488, 61000, 58000, 49152)]).astype(np.float16)
    x = x if axis == 1 else np.ascontiguousarray(x.T)
    scale = 2.0 ** 8 if fmt == "nvfp4" else 1.0
    want = rm.block_values(x, fmt, axis, scale)
    assert np.abs(want).max() > 65504
    assert np.array_equal(round_trip(ng, x, fmt, axis, scale), np.clip(want, -65504, 65504).astype(np.float16))
    assert np.array_equal(round_trip(ng, x, fmt, axis, scale, np.float32), want.astype(np.float32))


def test_nvfp4_scales_saturate_and_never_vanish(ng):
    x = np.zeros((4, 32), np.float32)
    x[0, :16] = np.linspace(0, 6 * 448 * 3.0, 16)       # scale limited to 448: numbers to 6 * 448
    x[1, :16] = np.linspace(0, 6 * 2.0 ** -12, 16)      # scale kept at 2^-9
    x[2, 16:] = 1.0
    for t in (1.0, 2.0 ** -32, 2.0 ** 32, 2.0 ** -8):
        got = round_trip(ng, x, "nvfp4", 1, t)
        assert np.array_equal(got.astype(np.float64), rm.block_values(x, "nvfp4", 1, t)), t


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("axis", [0, 1])
def test_infinities_and_nan_take_their_block_along(ng, fmt, axis):
    rng = np.random.default_rng(5)
    x = values(rng, (64, 96), np.float16)
    for (r, c), v in {(3, 5): np.inf, (17, 40): -np.inf, (50, 95): np.nan, (0, 64): np.inf}.items():
        x[r, c] = v
    want = rm.block_values(x, fmt, axis)
    for dtype in (np.float16, np.float32):
        got = round_trip(ng, x, fmt, axis, out_dtype=dtype)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)].astype(dtype))
    assert 0 < np.isnan(want).sum() < 200


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_views_of_any_strides(ng, fmt, axis, dtype):
    """Column slices at odd addresses, steps, transposed and reversed views; what lies around them stays."""
    rng = np.random.default_rng(11)
    x = values(rng, (90, 150), dtype)
    A = ng.array(x, dtype=dtype)
    cuts = [(slice(0, 70), slice(3, 104)), (slice(1, 90, 2), slice(0, 150, 3)), (slice(None), slice(8, 72)),
            (slice(None, None, -1), slice(5, 6)), (slice(10, 11), slice(None))]
    for rs, cs in cuts:
        for trans in (False, True):
            v, V = x[rs, cs], A[rs, cs]
            O = ng.array(np.full_like(x, 9.0), dtype=dtype)
            W = O[rs, cs]
            if trans:
                v, V, W = v.T, V.T, W.T
            Q = ng.block_empty(v.shape, fmt, axis=axis)
            ng.dequantize(ng.quantize(V, Q), W)
            want = np.full_like(x, 9.0)
            (want[rs, cs].T if trans else want[rs, cs])[...] = rm.block_values(v, fmt, axis).astype(dtype)
            assert np.array_equal(O.get(), want), (rs, cs, trans)


def test_several_matrices_from_one_call_and_the_same_buffer_again(ng):
    rng = np.random.default_rng(3)
    x = values(rng, (150, 70))
    q4, q8, w4 = (ng.block_empty(x.shape, f, axis=a) for f, a in (("mxfp4", 0), ("mxfp8", 1), ("nvfp4", 0)))
    outs = ng.quantize(ng.array(x), q4, q8, w4)
    assert outs == (q4, q8, w4)
    for data in (x, values(rng, x.shape)):          # no trace of the first matrix in the second's blocks
        ng.quantize(ng.array(data), q4, q8, w4)
        for q in outs:
            got = ng.dequantize(q, ng.empty(x.shape, dtype=np.float32)).get()
            assert np.array_equal(got, rm.block_values(data, q.format, q.axis))
            t = ng.dequantize(q.T, ng.empty(x.shape[::-1], dtype=np.float32)).get()
            assert np.array_equal(t, got.T) and q.T.T.axis == q.axis


@pytest.mark.parametrize("shape", [(130, 70), (20, 300), (1, 1), (65, 256)])
def test_padding_stays_zero(ng, shape):
    """Products read whole tiles of codes and scales: what lies behind a row's or the matrix's end is zero."""
    x = np.full(shape, 3.0, np.float16)
    for fmt in ("mxfp4", "nvfp4"):
        for axis in (0, 1):
            q = filled(ng, x if axis else x.T, fmt, axis)
            codes, scales = q.codes.get(), q.scales.get()
            odd = shape[1] % 2 * shape[0]
            assert (codes != 0).sum() == shape[0] * ((shape[1] + 1) // 2) and ((codes >> 4) != 0).sum() == (codes != 0).sum() - odd
            assert (scales != 0).sum() == shape[0] * -(-shape[1] // (16 if fmt == "nvfp4" else 32))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("shape", [(1, 1), (7, 33), (64, 128), (130, 257), (700, 3), (500, 17), (300, 48), (301, 70)])
def test_relu_mask_is_that_of_the_activation(ng, dtype, axis, shape):
    """Numbers far below their block's largest keep their sign, and so do those beside infinities and NaN; deltas
    that are infinite or NaN go where the activation was not positive."""
    rng = np.random.default_rng(shape[1])
    x = np.maximum(values(rng, shape, np.float16, 3.0), 0)
    if shape[1] > 8 and shape[0] > 6:
        x[2, 3], x[2, 4], x[5, 7], x[6, 7], x[6, 8] = 65504, 6e-8, np.inf, np.nan, -1.0
    e = rng.standard_normal(shape).astype(dtype)
    if x.size > 100:
        e[0, :9] = np.nan
        e[1, :9] = np.inf
    want = np.where(x > 0, e, 0)
    E = ng.array(e, dtype=dtype)
    got = ng.relu_mask(filled(ng, x, "mxfp8", axis), E).get()
    assert np.array_equal(got, want, equal_nan=True)
    wide = ng.array(np.full((shape[0] + 1, shape[1] + 3), 5.0), dtype=dtype)
    view = wide[1:, 2:shape[1] + 2]
    view[:] = ng.array(np.nan_to_num(e, nan=1.0, posinf=2.0), dtype=dtype)
    ng.relu_mask(filled(ng, x, "mxfp8", axis), view)
    full = np.full(wide.shape, 5.0)
    full[1:, 2:-1] = np.where(x > 0, np.nan_to_num(e, nan=1.0, posinf=2.0), 0)
    assert np.array_equal(wide.get(), full.astype(dtype))


# ---- products ----------------------------------------------------------------------------------------
def operands(rng, fmt, m, n, k):
    W = (rng.standard_normal((m, k)) * np.exp(0.5 * rng.standard_normal((m, 1)))).astype(np.float16)
    X = np.maximum(rng.standard_normal((k, n)), 0).astype(np.float16)
    return W, X


SIZES = [(1, 1, 1), (1, 1, 16), (3, 5, 33), (16, 1, 256), (128, 128, 256), (130, 17, 300), (257, 33, 1000), (1001, 125, 4097),
         (64, 300, 513), (200, 129, 64), (384, 65, 2048), (5, 1000, 640), (1, 4096, 512), (4096, 1, 4096), (640, 520, 768), (2500, 2304, 512), (2049, 2101, 1030), (2304, 2048, 2300)]


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_block_dot(ng, fmt, m, n, k):
    rng = np.random.default_rng(m + 7 * n + 13 * k)
    W, X = operands(rng, fmt, m, n, k)
    sw, sx = (2.0 ** -2, 2.0 ** -4) if fmt == "nvfp4" else (1.0, 1.0)
    A, B = filled(ng, W, fmt, 1, sw), filled(ng, X, fmt, 0, sx)
    a, b = rm.block_values(W, fmt, 1, sw), rm.block_values(X, fmt, 0, sx)
    ref, mag = a @ b, np.abs(a) @ np.abs(b)
    C = ng.empty((m, n))
    C.fill(np.nan)
    assert ng.block_dot(A, B, C) is C
    assert_close(C.get(), ref, product_tol(ref, mag, k), "fp16")
    F = ng.empty((m, n), dtype=np.float32)
    ng.block_dot(A, B, F)
    assert_close(F.get(), ref, product_tol(ref, mag, k, f32=True), "fp32")
    first = F.get()
    ng.block_dot(A, B, F)
    assert np.array_equal(first, F.get())


@pytest.mark.parametrize("m,n,k", [(70, 50, 100), (200, 300, 513), (9, 700, 96), (256, 128, 1024), (2100, 2061, 300)])
@pytest.mark.parametrize("mixed", [False, True])
def test_product_output_stage(ng, m, n, k, mixed):
    """alpha, ReLU, what is added to, rounding to nearest and stochastically, rows inside a wider matrix."""
    rng = np.random.default_rng(m + n)
    W, X = operands(rng, "mxfp4", m, n, k)
    W *= np.float16(0.25)
    if mixed:
        A, B = ng.array(W), filled(ng, np.ascontiguousarray(X.T), "mxfp8", 1).T
        a, b = W.astype(np.float64), rm.block_values(X, "mxfp8", 0)
    else:
        A, B = filled(ng, W, "mxfp4", 1), filled(ng, X, "mxfp4", 0)
        a, b = rm.block_values(W, "mxfp4", 1), rm.block_values(X, "mxfp4", 0)
    dot, mag = a @ b, np.abs(a) @ np.abs(b)
    old = rng.standard_normal((m, n)).astype(np.float16)
    ref = np.maximum(0.5 * dot, 0) - 2.0 * old
    sums = 0.5 * mag + 2.0 * np.abs(old)
    for dtype in (np.float16, np.float32):
        C = ng.array(old, dtype=dtype)
        ng.block_dot(A, B, C, alpha=0.5, beta=-2.0, relu=True)
        assert_close(C.get(), ref, product_tol(ref, sums, k + 2, f32=dtype is np.float32), str(dtype))
        wide = ng.array(np.full((m + 2, n + 5), 3.0), dtype=dtype)
        for c0 in (3, 0):           # at an odd address, and aligned with rows that are not
            view = wide[1:m + 1, c0:c0 + n]
            ng.block_dot(A, B, view, relu=True)
        got = wide.get()
        r1 = np.maximum(dot, 0)
        assert_close(got[1:m + 1, :n], r1, product_tol(r1, mag, k, f32=dtype is np.float32), "view")
        assert (got[0] == 3).all() and (got[m + 1] == 3).all() and (got[1:m + 1, n + 3:] == 3).all()
    C = ng.empty((m, n))
    r = ng.rand_state.offset
    ng.block_dot(A, B, C, stochastic_round=True)
    assert ng.rand_state.offset == r + 1
    got = C.get()
    assert_close(got, dot, product_tol(dot, mag, k, steps=2.0), "stochastic")
    ng.block_dot(A, B, C, stochastic_round=10)
    again = C.get()
    # other random bits, other roundings, where there is anything to round (a short sum of 4-bit numbers times powers
    # of two can be an fp16 number as it is: 9 x 700 x 96 has no other)
    between = dot.astype(np.float16) != dot
    assert (got != again)[between].any() or between.sum() < 100
    ng.rand_state.offset = r
    ng.block_dot(A, B, C, stochastic_round=10)
    assert np.array_equal(C.get(), got)


@pytest.mark.parametrize("m,n,k", [(300, 7, 40), (2049, 2301, 300), (2500, 2310, 96), (130, 13, 256)])
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_rows_that_end_inside_16_bytes_of_a_wider_matrix(ng, m, n, k, mixed, dtype):
    """Aligned rows with a ragged end: what lies behind them stays."""
    W, X = np.ones((m, k), np.float16), np.ones((k, n), np.float16)
    A = ng.array(W) if mixed else filled(ng, W, "mxfp4", 1)
    B = filled(ng, X, "mxfp8" if mixed else "mxfp4", 0)
    ld = -(-(n + 1) // 8) * 8
    wide = ng.array(np.full((m + 1, ld), 3.0), dtype=dtype)
    want = np.full((m + 1, ld), 3.0)
    for beta in (0.0, 1.0):
        ng.block_dot(A, B, wide[:m, :n], beta=beta)
        want[:m, :n] = k * (1 + beta)
        assert np.array_equal(wide.get(), want.astype(dtype)), beta


def long_matrix(ng, rows, cols, rng):
    """More than 2^32 numbers: zeros but for whole numbers up to 4 in the last two rows (read back as they are in every
    format whose blocks hold them: each block of 16 has a 4, and a 1 or 2 else)."""
    A = ng.empty((rows, cols), dtype=np.float16)
    A.fill(0)
    last = rng.choice([1.0, 2.0], (2, cols)).astype(np.float16)
    last[:, ::16] = 4
    A[rows - 2:].set(last)
    return A, last


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("axis", [0, 1])
def test_matrices_of_more_numbers_than_32_bits_count(ng, fmt, axis):
    rows, cols = 70002, 65008
    A, last = long_matrix(ng, rows, cols, np.random.default_rng(3))
    Q = ng.quantize(A, ng.block_empty((rows, cols), fmt, axis=axis))
    A.fill(9)
    ng.dequantize(Q, A)
    assert np.array_equal(A[rows - 2:].get(), last)
    assert not A[rows - 200:rows - 2].get().any()
    if fmt == "mxfp8" and axis == 1:
        A.fill(9)
        ng.relu_mask(Q, A)
        assert np.array_equal(A[rows - 2:].get(), np.where(last > 0, 9.0, 0.0))
        assert not A[rows - 200:rows - 2].get().any()


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_products_of_long_matrices(ng, fmt):
    """The long matrix as the left side, and as the output. Sums of up to 65008 products of up to 4, whole numbers below
    2^24, are exact in 32 bits."""
    rows, cols = 70002, 65008
    A, last = long_matrix(ng, rows, cols, np.random.default_rng(4))
    X = np.ones((8, cols), np.float16)
    B = ng.quantize(ng.array(X), ng.block_empty((8, cols), fmt)).T
    left = A if fmt == "mxfp8" else ng.quantize(A, ng.block_empty((rows, cols), fmt))
    C = ng.empty((rows, 8), dtype=np.float32)
    ng.block_dot(left, B, C)
    got = C.get()
    assert not got[:-2].any()
    assert np.array_equal(got[-2:], np.tile(last.sum(axis=1, dtype=np.float64)[:, None], (1, 8)))

    w = np.zeros((rows, 32), np.float16)
    w[-2:] = 1
    x = np.ones((cols, 32), np.float16)
    x[-1] = 2
    W = ng.array(w) if fmt == "mxfp8" else filled(ng, w, fmt, 1)
    A.fill(9)
    ng.block_dot(W, filled(ng, x, fmt, 1).T, A)
    assert not A[rows - 200:rows - 2].get().any()
    assert np.array_equal(A[rows - 2:].get(), np.tile(32 * x[:, 0], (2, 1)))


@pytest.mark.parametrize("m,n,k", [(5, 40, 7), (300, 300, 45), (130, 700, 1003), (2100, 2061, 301)])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4", "nvfp4"])
def test_what_lies_around_an_input_is_not_read(ng, m, n, k, fmt):
    """Inputs that are views of wider matrices, aligned or not, between NaN. In nvfp4 a block of ones has the scale
    1/6, to the nearest e4m3 number 0.171875, and 1 is read back as 6 * 0.171875 = 1.03125; its square is a multiple of
    2^-10 and sums of up to 2^13 of them are exact in 32 bits."""
    one = 1.03125 if fmt == "nvfp4" else 1.0
    for first, more in ((0, -k % 8), (8, -k % 8), (1, 2)):
        def within(r, c):
            wide = np.full((r + 2, first + c + more), np.nan, np.float16)
            wide[1:r + 1, first:first + c] = 1
            return ng.array(wide)[1:r + 1, first:first + c]
        W, X = within(m, k), within(n, k)
        A = W if fmt == "mxfp8" else ng.quantize(W, ng.block_empty((m, k), fmt))
        B = ng.quantize(X, ng.block_empty((n, k), fmt)).T
        C = ng.empty((m, n), dtype=np.float32)
        ng.block_dot(A, B, C)
        assert np.array_equal(C.get(), np.full((m, n), k * one * one)), (first, more)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (2, 3, 31), (128, 64, 32), (33, 17, 125), (130, 257, 300), (1001, 515, 125),
                                   (64, 256, 2048), (300, 200, 64), (16, 1000, 128), (257, 9, 4100),
                                   (2048, 1301, 70), (2496, 2304, 96), (2400, 2311, 33), (19000, 65, 40)])
@pytest.mark.parametrize("shift", [0, 1])
def test_block_dot_f16(ng, m, n, k, shift):
    """The weight gradient: plain fp16 deltas (also at odd addresses and in rows of a wider matrix) with an 8-bit record."""
    rng = np.random.default_rng(m + n + k)
    E = (rng.standard_normal((m, k)) * 0.05).astype(np.float16)
    X = np.maximum(values(rng, (n, k)), 0)
    wide = np.zeros((m, k + 2 * shift), np.float16)
    wide[:, shift:shift + k] = E
    dE = ng.array(wide)[:, shift:shift + k]
    B = filled(ng, X, "mxfp8", 1).T
    a, b = E.astype(np.float64), rm.block_values(X, "mxfp8", 1).T
    ref, mag = a @ b, np.abs(a) @ np.abs(b)
    C, F = ng.empty((m, n)), ng.empty((m, n), dtype=np.float32)
    assert_close(ng.block_dot(dE, B, C).get(), ref, product_tol(ref, mag, k), "fp16")
    assert_close(ng.block_dot(dE, B, F).get(), ref, product_tol(ref, mag, k, f32=True), "fp32")
    # against differences: sum(E * (W X)) is linear in W, and its derivative is the gradient
    W = np.zeros((m, n))
    i, j = m // 2, n // 3
    f = lambda w: float((a * (w @ b.T if b.shape[0] != n else w @ b)).sum())
    W[i, j] = 1.0
    assert abs(f(W) - float(F.get()[i, j])) <= product_tol(ref, mag, k, f32=True)[i, j] + 1e-12 * mag[i, j]


@pytest.mark.parametrize("m,n,k", [(1, 3, 700), (70, 90, 1000), (130, 65, 2049), (129, 200, 1537), (300, 300, 1500), (513, 20, 650)])
@pytest.mark.parametrize("aligned", [False, True])
def test_long_sums_of_few_outputs(ng, m, n, k, aligned):
    """Sums that are split over several SMs: every output form, views, and the same bits every time."""
    rng = np.random.default_rng(m + n + k)
    E = (rng.standard_normal((m, k)) * 0.1).astype(np.float16)
    X = np.maximum(rng.standard_normal((n, k)), 0).astype(np.float16)
    lda = k + -k % 8 if aligned else k + 1 + k % 2
    wide = np.full((m, lda), np.nan, np.float16)
    wide[:, :k] = E
    A, B = ng.array(wide)[:, :k], ng.quantize(ng.array(X), ng.block_empty((n, k), "mxfp8")).T
    x = rm.block_values(X, "mxfp8")
    e = E.astype(np.float64)
    dot, mag = e @ x.T, np.abs(e) @ np.abs(x).T
    ldc = n + -n % 8 if aligned else n + 3
    for dtype in (np.float16, np.float32):
        old = rng.standard_normal((m, n)).astype(np.float16)
        first = None
        for _ in range(3):
            C = ng.array(np.full((m + 1, ldc), 7.0), dtype=dtype)
            C[:m, :n] = ng.array(old, dtype=dtype)
            ng.block_dot(A, B, C[:m, :n], alpha=2.0, beta=-1.0, relu=True)
            got = C.get()
            first = got if first is None else first
            assert np.array_equal(first, got)
        ref = np.maximum(2 * dot, 0) - old
        assert_close(got[:m, :n], ref, product_tol(ref, 2 * mag + np.abs(old), k + 2, f32=dtype is np.float32), str(dtype))
        assert (got[m] == 7).all() and (got[:, n:] == 7).all()
    C = ng.empty((m, n))
    ng.block_dot(A, B, C, stochastic_round=10)
    assert_close(C.get(), dot, product_tol(dot, mag, k, steps=2.0))


def test_extreme_records_in_the_mixed_product(ng):
    """The largest and smallest fp16 numbers, and numbers that a record keeps only by their sign."""
    X = np.zeros((8, 64), np.float16)
    X[0, :4] = 65504, 60000, 1e-3, 6e-8
    X[1, :3] = 6e-8, 1.2e-7, 1.8e-7
    X[2, 32:36] = 1e-4, 6.1e-5, 3e-5, 6e-8
    X[3] = np.linspace(0, 1, 64)
    E = np.eye(64, dtype=np.float16)
    F = ng.empty((64, 8), dtype=np.float32)
    ng.block_dot(ng.array(E), filled(ng, X, "mxfp8", 1).T, F)
    want = rm.block_values(X, "mxfp8", 1)
    assert want[0, 0] == 65536          # what 65504 is rounded to counts as fp16's largest number
    assert np.array_equal(F.get(), np.minimum(want, 65504).T)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "mxfp8"])
def test_infinities_and_nan_reach_what_they_meet(ng, fmt):
    """An operand's row with an infinity or NaN gives NaN in its row (column) of the product and nowhere else."""
    rng = np.random.default_rng(2)
    m, n, k = 140, 36, 300
    W, X = operands(rng, fmt, m, n, k)
    if fmt == "mxfp8":
        W[7, 150] = np.nan
        A = ng.array(W)
        a = W.astype(np.float64)
    else:
        W[7, 150], W[133, 299] = np.inf, np.nan
        A = filled(ng, W, fmt, 1)
        a = rm.block_values(W, fmt, 1)
    X[290, 20] = -np.inf
    B, b = filled(ng, X, fmt, 0), rm.block_values(X, fmt, 0)
    C = ng.empty((m, n))
    got = ng.block_dot(A, B, C).get()
    bad_rows = [7] if fmt == "mxfp8" else [7, 133]
    want = np.zeros((m, n), bool)
    want[bad_rows] = True
    want[:, 20] = True
    assert np.array_equal(np.isnan(got), want)
    ok = ~want
    ref = np.nan_to_num(a) @ np.nan_to_num(b)
    mag = np.abs(np.nan_to_num(a)) @ np.abs(np.nan_to_num(b))
    assert (np.abs(got - ref)[ok] <= product_tol(ref, mag, k)[ok]).all()


def test_other_streams_and_recorded_sequences():
    """A whole run of them (quantise, product, record, mask, gradient) live, on a stream of its own, and replayed with
    other inputs in the same buffers; two recordings of the same stream in turn."""
    ng = NervanaGPU(stochastic_round=False)
    ng.stream = ng.new_stream()
    rng = np.random.default_rng(8)
    m, n, k = 192, 72, 320
    W = (rng.standard_normal((m, k)) * 0.1).astype(np.float16)
    W4 = filled(ng, W, "nvfp4", 1, 2.0 ** -6)
    X, E, D = ng.empty((k, n)), ng.empty((m, n)), ng.empty((k, n))
    X4, X8 = ng.block_empty((k, n), "nvfp4", axis=0), ng.block_empty((k, n), "mxfp8")
    Y, dW = ng.empty((m, n)), ng.empty((m, k), dtype=np.float32)

    def step():
        ng.quantize(X, X4, X8)
        ng.block_dot(W4, X4, Y, relu=True)
        ng.block_dot(E, X8.T, dW)
        ng.relu_mask(X8, D)

    def check(seed):
        r = np.random.default_rng(seed)
        x = np.maximum(r.standard_normal((k, n)), 0).astype(np.float16)
        e, d = (0.1 * r.standard_normal(s).astype(np.float16) for s in ((m, n), (k, n)))
        X.set(x), E.set(e), D.set(d)
        yield
        a, b = rm.block_values(W, "nvfp4", 1, 2.0 ** -6), rm.block_values(x, "nvfp4", 0)
        ref = np.maximum(a @ b, 0)
        assert_close(Y.get(), ref, product_tol(ref, np.abs(a) @ b, k))
        x8 = rm.block_values(x, "mxfp8", 1)
        ref = e.astype(np.float64) @ x8.T
        assert_close(dW.get(), ref, product_tol(ref, np.abs(e.astype(np.float64)) @ x8.T, n, f32=True))
        assert np.array_equal(D.get(), np.where(x > 0, d, 0))

    for _ in check(1):
        step()
    first, second = ng.capture(step), ng.capture(step)
    for seed, run in enumerate((first, second, first, step, second), 10):
        for _ in check(seed):
            run.launch() if run is not step else step()
    first.release()
    for _ in check(30):
        second.launch()


def test_a_long_sum_recorded_without_room_and_with_it():
    """600 x 500 x 8200 would take a copy in scratch memory: a recording on a new stream, which cannot grow it, and one after
    a run that did; two recordings in turn."""
    ng = NervanaGPU(stochastic_round=False)
    rng = np.random.default_rng(5)
    m, n, k = 600, 500, 8200
    E = (rng.standard_normal((m, k)) * 0.1).astype(np.float16)
    X = np.maximum(rng.standard_normal((n, k)), 0).astype(np.float16)
    A, Q = ng.array(E), ng.quantize(ng.array(X), ng.block_empty((n, k), "mxfp8"))
    ng.synchronize()
    x, e = rm.block_values(X, "mxfp8"), E.astype(np.float64)
    ref, mag = e @ x.T, np.abs(e) @ x.T
    ng.stream = ng.new_stream()
    C, D = ng.zeros((m, n), dtype=np.float32), ng.zeros((m, n), dtype=np.float32)
    first = ng.capture(lambda: ng.block_dot(A, Q.T, C))
    first.launch()
    assert_close(C.get(), ref, product_tol(ref, mag, k, f32=True))
    ng.block_dot(A, Q.T, C)
    second = ng.capture(lambda: ng.block_dot(A, Q.T, D))
    for run in (second, first, second):
        C.fill(0), D.fill(0)
        run.launch()
        assert_close((D if run is second else C).get(), ref, product_tol(ref, mag, k, f32=True))


def test_launches_and_no_fallback(ng, lib):
    """Each call launches the library's kernels and none of the CUDA-core products."""
    import ctypes
    rng = np.random.default_rng(1)
    W, X = operands(rng, "nvfp4", 256, 128, 512)
    A, B, X8 = filled(ng, W, "nvfp4", 1), filled(ng, X, "nvfp4", 0), filled(ng, X, "mxfp8", 1)
    C, dX = ng.empty((256, 128)), ng.empty((256, 512))
    n0, f0, n1, f1 = (ctypes.c_ulonglong() for _ in range(4))
    lib.ng_launch_count(ctypes.byref(n0)), lib.ng_fallback_launch_count(ctypes.byref(f0))
    ng.block_dot(A, B, C)
    ng.block_dot(C, X8.T, dX)
    lib.ng_launch_count(ctypes.byref(n1)), lib.ng_fallback_launch_count(ctypes.byref(f1))
    assert n1.value - n0.value >= 2 and f1.value == f0.value
    ng.synchronize()


def test_device_memory_of_another_device_is_refused(ng):
    q = ng.block_empty((4, 4), "mxfp8")
    q.desc.device += 1
    with pytest.raises(_lib.NervanaError, match="current device"):
        ng.quantize(ng.zeros((4, 4)), q)
