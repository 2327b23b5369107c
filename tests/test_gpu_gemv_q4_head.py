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


GATED = 1025 * 16   # pairs of tiles with SwiGLU


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 16, 17, 24, 32])
@pytest.mark.parametrize("epi,norm", [(0, False), (0, True), (1, False), (1, True)])
@pytest.mark.parametrize("k,group", [(1024, 32), (2048, 128)])
def test_epilogues_and_norm(qa, rows, epi, norm, k, group):
    """Every number of waves that share a row of x, one and two parts of the rows, joins of several waves."""
    rng = np.random.default_rng(rows + epi)
    q, d = matrix(OUT, k, group)
    x = (rng.standard_normal((rows, k)) * 3).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32) if norm else None
    y0 = rng.standard_normal((rows, OUT)).astype(np.float32) if epi == 1 else None
    close(gemv(qa, q, d, x, group, epi, w, y0), *plain(q, d, x, epi, w, y0))


@pytest.mark.parametrize("rows", [1, 3, 8, 14, 20, 32])
@pytest.mark.parametrize("norm", [False, True])
def test_gated(qa, rows, norm):
    rng = np.random.default_rng(rows)
    k, group = 1024, 64
    q, d = matrix(2 * GATED, k, group)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32) if norm else None
    close(gemv(qa, q, d, x, group, 2, w), *plain(q, d, x, 2, w), rel=8e-6)


@pytest.mark.parametrize("k", [128, 384, 2048, 4096, 16384])
@pytest.mark.parametrize("rows", [1, 2, 4])
def test_few_rows_of_any_width(qa, rows, k):
    """Up to 2048 columns for each of the 8 waves of one row, 4 of two and 2 of four; wider rows are split by each wave."""
    out = OUT if k <= 4096 else 1025 * 16
    rng = np.random.default_rng(k + rows)
    q, d = weights(rng, out, k, 128)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    close(gemv(qa, q, d, x, 128, 0, w), *plain(q, d, x, 0, w), rel=2e-6 if k <= 6144 else 3e-6)


@pytest.mark.parametrize("rows,norm", [(1, True), (8, True), (16, False), (32, True)])
def test_vocabulary_of_the_larger_model(qa, rows, norm):
    """151936 x 2048, of which every result of 120 rows of W, the first and the last ones among them, is compared."""
    out, k, group = 151936, 2048, 64
    rng = np.random.default_rng(rows)
    words = rng.integers(0, 2 ** 32, (out // 16, k // 128, 4, 16, 4), np.uint32)     # tile, block, j, row, word
    d = (0.002 + 0.006 * rng.random((out // 16, k // group, 16), np.float32)).astype(np.float16)
    x = (rng.standard_normal((rows, k)) * 2).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32) if norm else None
    dev = qa.DeviceArray.from_numpy
    y, bufs, dw = dev(np.full((rows + 1, out), 9.5, np.float32)), [dev(words), dev(d), dev(x)], dev(w) if norm else None
    print(f"head rows={rows} norm={norm}", flush=True)
    qa.check(qa.lib.qa_gemv_q4(bufs[0].ptr, bufs[1].ptr, group, out, k, bufs[2].ptr, rows, y.ptr, 0, dw.ptr if norm else None, 1e-6, None))
    qa.synchronize()
    got = y.numpy()
    assert (got[rows] == 9.5).all() and np.isfinite(got).all()
    pick = np.unique(np.r_[0:16, out - 16:out, rng.integers(0, out, 90)])
    of = words[pick // 16, :, :, pick % 16]                                           # row, block, j, word
    q = np.stack([of >> np.uint32(4 * (e // 2) + 16 * (e % 2)) & 15 for e in range(8)], -1)
    q = q.transpose(0, 1, 3, 2, 4).reshape(len(pick), k)                              # row, block, word, j, e: in order of column
    close(got[:rows, pick], *plain(q, d[pick // 16, :, pick % 16], x, 0, w))


@pytest.mark.parametrize("rows", [1, 2, 6, 14, 30])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e5, 1e30])
def test_magnitudes_of_x(qa, rows, scale, norm):
    """Rows of unlike size side by side, each with its own power of two."""
    rng = np.random.default_rng(rows)
    k, group = 1024, 32
    q, d = matrix(OUT, k, group)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    x[::2] *= np.float32(scale)
    w = np.ones(k, np.float32) if norm else None
    got = gemv(qa, q, d, x, group, 0, w).astype(np.float64)
    want, _ = plain(q, d, x, 0, w)
    for r in range(rows):
        assert np.linalg.norm(got[r] - want[r]) <= 2e-6 * np.linalg.norm(want[r]), (r, scale)


@pytest.mark.parametrize("rows", [1, 2, 8, 16])
@pytest.mark.parametrize("norm", [False, True])
def test_outliers_in_x(qa, rows, norm):
    """One value 2^20 times the others, on a column of zero weights: the rest keeps its bits.  The row is split in units of
    2^6 (2^20 goes to 2^14); second parts below 2^-14 of a unit are f16 subnormals, off by at most 2^-25 of it: 2^-19 for each
    x, times the factor of RMSNorm, over all weights."""
    rng = np.random.default_rng(5)
    k, group = 1024, 32
    q, d = matrix(OUT, k, group)
    q = q.copy()
    q[:, 7] = 8
    x = rng.standard_normal((rows, k)).astype(np.float32)
    x[0, 7] = 2.0 ** 20
    w = np.ones(k, np.float32) if norm else None
    got = gemv(qa, q, d, x, group, 0, w)
    want, size = plain(q, d, x, 0, w)
    f = 1 / np.sqrt((x[0].astype(np.float64) ** 2).mean()) if norm else 1.0
    assert np.linalg.norm(got[0] - want[0]) <= 2e-6 * np.linalg.norm(want[0]) + 2.0 ** -19 * f * np.linalg.norm(values(q, d))
    if rows > 1:
        close(got[1:], want[1:], size[1:])


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("rows", [1, 2, 4, 8, 16, 20])
@pytest.mark.parametrize("norm", [False, True])
def test_not_finite_x(qa, rows, norm, value):
    """An infinity stays one (NaN where its weight is 0, and behind the norm, whose factor is 0), NaN stays NaN, in its row."""
    rng = np.random.default_rng(6)
    k, group, at = 2048, 128, 1301
    q, d = matrix(OUT, k, group)
    q = q.copy()
    q[:16, at], q[16:31, at], q[31, at] = 12, 3, 8
    x = rng.standard_normal((rows, k)).astype(np.float32)
    x[rows // 2, at] = value
    w = np.ones(k, np.float32) if norm else None
    got = gemv(qa, q, d, x, group, 0, w)
    bad = got[rows // 2]
    if norm or np.isnan(value):
        assert np.isnan(bad).all()
    else:
        assert (bad[:16] == value).all() and (bad[16:31] == -value).all()
        np.testing.assert_array_equal(bad, np.where(q[:, at] == 8, np.nan, np.where(q[:, at] > 8, value, -value)))
    rest = [r for r in range(rows) if r != rows // 2]
    if rest:
        want, size = plain(q, d, x[rest], 0, w)
        close(got[rest], want, size)
