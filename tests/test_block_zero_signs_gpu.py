"""Signs of zeros in matrices in blocks (B200 only): every form of a quantisation writes the same bytes. (In nvfp4 the signs of
zeros, which that format does not promise, may depend on whether the numbers came as fp16 or fp32.)"""
import numpy as np
import pytest

from nervanagpu_b200 import NervanaGPU  # noqa: F401  (the ng fixture's class)

pytestmark = pytest.mark.gpu


def numbers(outer, inner):
    """Fp16 numbers with zeros of both signs, numbers that their block's scale rounds to zero, blocks of such zeros only, and blocks
    so small that their factor is beyond 2^30."""
    rng = np.random.default_rng(outer + inner)
    x = rng.standard_normal((outer, inner)).astype(np.float16)
    x[rng.random(x.shape) < 0.2] = 0.0
    x[rng.random(x.shape) < 0.2] = -0.0
    tiny = rng.random(x.shape) < 0.2
    x[tiny] = np.where(rng.random(x.shape) < 0.5, -6e-8, 6e-8).astype(np.float16)[tiny]
    x[1] = np.where(rng.random(inner) < 0.5, -0.0, 0.0)
    x[2] = np.where(rng.random(inner) < 0.5, -6e-8, -0.0)
    x[3, :] = -0.0
    return x


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "mxfp8"])
@pytest.mark.parametrize("inner", [5, 16, 40, 96, 300])
def test_the_same_numbers_give_the_same_codes_in_every_form(ng, fmt, inner):
    outer = 130
    x = numbers(outer, inner)
    ld = inner + -inner % 16
    forms = {}
    for dtype in (np.float16, np.float32):
        v = x.astype(dtype)
        wide = np.full((outer, ld), 3, dtype)
        wide[:, :inner] = v
        forms["rows", dtype] = ng.array(wide, dtype=dtype)[:, :inner], 1
        odd = np.full((outer, ld + 3), 3, dtype)
        odd[:, 1:inner + 1] = v
        forms["rows at odd addresses", dtype] = ng.array(odd, dtype=dtype)[:, 1:inner + 1], 1
        t = np.ascontiguousarray(v.T)
        forms["columns", dtype] = ng.array(t, dtype=dtype), 0
        odd = np.full((inner, outer + 3), 3, dtype)
        odd[:, 1:outer + 1] = t
        forms["columns at odd addresses", dtype] = ng.array(odd, dtype=dtype)[:, 1:outer + 1], 0
        step = np.full((inner, 2 * outer), 3, dtype)
        step[:, ::2] = t
        forms["columns two apart", dtype] = ng.array(step, dtype=dtype)[:, ::2], 0
    def without_signs_of_zeros(codes):
        lo, hi = codes & 15, codes >> 4
        return np.where(lo == 8, 0, lo) | np.where(hi == 8, 0, hi) << 4

    first = {}
    for what, (A, axis) in forms.items():
        Q = ng.quantize(A, ng.block_empty(A.shape, fmt, axis=axis))
        codes, scales = Q.codes.get(), Q.scales.get()
        if fmt != "nvfp4":
            group = None                # all forms
        else:
            group = what[1]             # those of one type; the others but for zeros
            for other, _ in first.values():
                assert np.array_equal(without_signs_of_zeros(codes), without_signs_of_zeros(other)), what
        want = first.setdefault(group, (codes, scales))
        assert np.array_equal(codes, want[0]) and np.array_equal(scales, want[1]), what
        for out in (np.float16, np.float32):
            got, signs = ng.dequantize(Q, ng.empty(A.shape, dtype=out)).get(), np.signbit(x if axis else x.T)
            checked = got != 0 if fmt == "nvfp4" else np.ones(got.shape, bool)
            assert np.array_equal(np.signbit(got)[checked], signs[checked]), (what, out)
