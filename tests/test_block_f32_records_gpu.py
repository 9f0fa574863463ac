"""Records made from fp32 numbers in the fp16 x mxfp8 product (B200 only)."""
import numpy as np
import pytest

from oracle import reference_math as rm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(40, 30, 64), (70, 90, 2048), (600, 500, 8200), (1000, 2000, 70)])
def test_a_record_counts_as_fp16_numbers(ng, m, n, k):
    """Values beyond 65504 count as that, those below fp16's normal range are rounded to it, whichever form the product takes (whole
    sums, sums in parts, a copy). Each row of E selects one number of every row of the record, so the results are these."""
    rng = np.random.default_rng(k)
    X = (rng.standard_normal((n, k)) * np.exp(6 * rng.standard_normal((n, 1)))).astype(np.float32)
    X[0] *= np.float32(1e30)
    X[1] = np.linspace(-1e-6, 1e-6, k)
    X[2, :32], X[2, 32:] = 1e-30, 7e4
    at = rng.integers(0, k, m)
    E = np.zeros((m, k), np.float16)
    E[np.arange(m), at] = 1
    Q = ng.quantize(ng.array(X, dtype=np.float32), ng.block_empty((n, k), "mxfp8"))
    F = ng.block_dot(ng.array(E), Q.T, ng.empty((m, n), dtype=np.float32)).get()
    want = np.clip(rm.block_values(X, "mxfp8"), -65504, 65504).astype(np.float16)
    assert (np.abs(want) == 65504).any() and (np.abs(want[1]) < 2.0 ** -14).all()
    assert np.array_equal(F, want[:, at].T.astype(np.float32))
