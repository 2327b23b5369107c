"""4-bit products of more than 1024 tiles of 16 rows (an LM head), whose x lies whole in LDS, against 64-bit sums.

The smallest such matrix is taken: 1025 tiles, the last one with rows that do not exist.  Statements, packing and tolerances are
those of test_gpu_gemv_q4.py (relative 2-norm 2e-6, with SwiGLU 8e-6; a value 2^-16 of the norm of its terms)."""
import functools

import numpy as np
import pytest

from test_gpu_gemv_q4 import close, gemv, plain, values, weights

pytestmark = pytest.mark.gpu

OUT = 1024 * 16 + 10


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


@functools.lru_cache(maxsize=2)
def matrix(out, k, group):
    return weights(np.random.default_rng(k + group), out, k, group)


def small_bar(w, factor):
    """What f32 cannot hold of a row of x far below 1 with factor `factor`: x times its norm weight is off by at most
    2^-150 where that is subnormal, in every column, and a result by as much again."""
    return 2.0 ** -150 * (factor * np.linalg.norm(w) + np.sqrt(len(w)))


@pytest.mark.parametrize("scale", [1e-40, 1e-36, 1e-33])
@pytest.mark.parametrize("out,rows", [(OUT, 1), (OUT, 2), (OUT, 4), (OUT, 8), (OUT, 16), (OUT, 32), (80, 1), (80, 8)])
def test_norm_of_small_x(qa, out, rows, scale):
    """RMSNorm's factor is 1000 for such rows (eps 1e-6): it does not meet the power of two that brings x to f16's range.
    Some columns are zero, and a row of ordinary size and one of zeros lie beside the small ones."""
    k, group = 1024, 64
    q, d = matrix(out, k, group)
    rng = np.random.default_rng(rows)
    x = (rng.standard_normal((rows, k)) * scale).astype(np.float32)
    x[:, ::5] = 0.0
    if rows > 2:
        x[1] = rng.standard_normal(k)
        x[2] = 0.0
    w = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    got = gemv(qa, q, d, x, group, 0, w).astype(np.float64)
    want, _ = plain(q, d, x, 0, w)
    assert np.isfinite(got).all()
    for r in range(rows):
        bar = small_bar(values(q, d), 1000.0) if 0 < np.abs(x[r]).max() < 1e-30 else 0.0
        assert np.linalg.norm(got[r] - want[r]) <= 2e-6 * np.linalg.norm(want[r]) + bar, r


@pytest.mark.parametrize("scale", [1e20, 1e30, 3e37])
@pytest.mark.parametrize("out,rows", [(OUT, 1), (OUT, 2), (OUT, 8), (OUT, 16), (80, 1), (80, 8), (80, 20)])
def test_norm_of_x_whose_squares_pass_f32(qa, out, rows, scale):
    """The mean of squares is no f32 from 1.8e19 on; the normalised row is as small as any."""
    k, group = 1024, 64
    q, d = matrix(out, k, group)
    rng = np.random.default_rng(rows)
    x = np.clip(rng.standard_normal((rows, k)), -5, 5).astype(np.float32) * np.float32(scale)
    if rows > 2:
        x[1] = rng.standard_normal(k)
    w = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    got = gemv(qa, q, d, x, group, 0, w)
    want, size = plain(q, d, x, 0, w)
    close(got, want, size)
