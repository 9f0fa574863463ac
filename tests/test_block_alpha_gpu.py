"""Factors of a 4-bit product at the ends of fp32 (B200 only)."""
import numpy as np
import pytest

from oracle import reference_math as rm
from tests._util import assert_close
from tests.test_blocks_gpu import product_tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(40, 24), (300, 280)])
def test_a_small_factor_and_scales_that_undo_each_other(ng, m, n):
    """2^-32 * 2^32 is 1: the factor counts as it is, also where one of them would take it below fp32's normal range."""
    rng = np.random.default_rng(m)
    k = 16
    W = (rng.standard_normal((m, k)) * 2.0 ** -32).astype(np.float32)
    X = (rng.standard_normal((k, n)) * 2.0 ** 32).astype(np.float32)
    A = ng.quantize(ng.array(W, dtype=np.float32), ng.block_empty((m, k), "nvfp4", scale=2.0 ** -32))
    B = ng.quantize(ng.array(X, dtype=np.float32), ng.block_empty((k, n), "nvfp4", axis=0, scale=2.0 ** 32))
    a, b = rm.block_values(W, "nvfp4", 1, 2.0 ** -32), rm.block_values(X, "nvfp4", 0, 2.0 ** 32)
    for alpha in (float(np.float32(1.2345678 * 2.0 ** -110)), float(np.float32(1.2345678 * 2.0 ** 100))):
        C = ng.empty((m, n), dtype=np.float32)
        ng.block_dot(A, B, C, alpha=alpha)
        # (in units of the factor's power of two, so that the comparison is in the normal range; the factor rounds once more)
        unit = 2.0 ** np.floor(np.log2(alpha))
        ref, mag = (alpha / unit) * (a @ b), (alpha / unit) * (np.abs(a) @ np.abs(b))
        assert_close((C.get().astype(np.float64) / unit).astype(np.float32), ref, product_tol(ref, mag, k + 2, f32=True), str(alpha))
