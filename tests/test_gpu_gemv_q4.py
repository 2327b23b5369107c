"""4-bit weights: the packed form against a plain quantiser, and matrix-vector products against 64-bit sums.

Tolerances.  Products are exact; a group's sum and the sum over groups are f32 sums of at most 128 and in_dim / 32 terms, of
random signs: the relative 2-norm error is below sqrt(in_dim / 32 + 128) 2^-24 = 1.1e-6 at 6144 columns, plus 2^-22 of the
split and 3 2^-24 of RMSNorm: 2e-6.  SwiGLU multiplies two of them and an exp: 8e-6.  A single value: 2^-16 of the norm of
its terms, sqrt(sum (w x)^2), about 250 of those roundings."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


def quantise(w, group):
    """(q 0..15 [out][in], d f16 [out][in / group]) of f32 rows."""
    g = w.reshape(len(w), -1, group)
    d = (np.abs(g).max(-1) / np.float32(7.0)).astype(np.float16)
    df = d.astype(np.float32)[..., None]
    with np.errstate(all="ignore"):
        q = np.where(df > 0, np.clip(np.rint(g / df), -8, 7), 0.0)
    return (q.reshape(w.shape) + 8).astype(np.uint32), d


def packed(q, d):
    """The packed words and scales of whole tiles."""
    out, k = q.shape
    pad = -(-out // 16) * 16
    qq = np.full((pad, k), 8, np.uint32)
    qq[:out] = q
    dd = np.zeros((pad, d.shape[1]), np.float16)
    dd[:out] = d
    words = np.zeros((pad // 16, k // 128, 4, 16, 4), np.uint32)      # tile, block, j, row, word
    v = qq.reshape(pad // 16, 16, k // 128, 4, 4, 8)                  # tile, row, block, word, j, e
    for e in range(8):
        words |= v[..., e].transpose(0, 2, 4, 1, 3) << np.uint32(4 * (e // 2) + 16 * (e % 2))
    return words.reshape(-1).view(np.uint8).copy(), np.ascontiguousarray(dd.reshape(pad // 16, 16, -1).transpose(0, 2, 1))


def values(q, d):
    group = q.shape[1] // d.shape[1]
    return (q.astype(np.float64) - 8) * np.repeat(d.astype(np.float64), group, 1)


@pytest.mark.parametrize("out,k,group", [(16, 128, 32), (1, 128, 128), (17, 256, 64), (100, 384, 32), (48, 1024, 128)])
def test_pack(qa, out, k, group):
    rng = np.random.default_rng(out)
    w = (rng.standard_normal((out, k)) * 0.02).astype(np.float32)
    w[0, :group] = 0.0
    w[-1, -group:] = 1e-9 * np.arange(group)              # the scale rounds to zero or a subnormal
    w[out // 2, 0] = 3e4
    w[0, -1], w[0, -2] = 0.07, -0.08
    q, d = quantise(w, group)
    want_w, want_d = packed(q, d)
    dw, ds = (qa.DeviceArray((n,), t) for n, t in ((qa.lib.qa_q4_weight_bytes(out, k), np.uint8), (qa.lib.qa_q4_scale_count(out, k, group), np.uint16)))
    src = qa.DeviceArray.from_numpy(w)
    qa.check(qa.lib.qa_pack_q4(src.ptr, out, k, group, dw.ptr, ds.ptr, None))
    qa.synchronize()
    np.testing.assert_array_equal(dw.numpy(), want_w)
    np.testing.assert_array_equal(ds.numpy(), want_d.reshape(-1).view(np.uint16))
    # half a step of the grid and the scale's own rounding (2^-11, and 2^-25 where it is subnormal) times 8 steps
    err, s = np.abs(values(q, d) - w), np.repeat(d.astype(np.float64), group, 1)
    assert (err <= s * (0.5 + 8 * 2.0 ** -11) + 8 * 2.0 ** -25).all()


def gemv(qa, q, d, x, group, epi=0, norm=None, y0=None, eps=1e-6):
    w, s = packed(q, d)
    rows, out = x.shape[0], q.shape[0] // (2 if epi == 2 else 1)
    y = np.full((rows + 1, out), 9.5, np.float32)
    if y0 is not None:
        y[:rows] = y0
    dv = [qa.DeviceArray.from_numpy(a) for a in (w, s, x, y)]
    dn = qa.DeviceArray.from_numpy(norm) if norm is not None else None
    print(f"q4 out={out} in={x.shape[1]} rows={rows} group={group} epilogue={epi} norm={norm is not None}", flush=True)
    qa.check(qa.lib.qa_gemv_q4(dv[0].ptr, dv[1].ptr, group, out, x.shape[1], dv[2].ptr, rows, dv[3].ptr, epi, dn.ptr if dn else None, eps, None))
    qa.synchronize()
    got = dv[3].numpy()
    assert (got[rows] == 9.5).all()
    return got[:rows]


def plain(q, d, x, epi=0, norm=None, y0=None, eps=1e-6):
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    w = values(q, d)
    y, size = x @ w.T, np.sqrt((x * x) @ (w * w).T)
    if epi == 1:
        return y + y0, size + np.abs(y0)
    if epi == 2:
        g, u = np.split(y, 2, 1)
        a, b = np.split(size, 2, 1)
        silu = g / (1 + np.exp(-g))
        return silu * u, (np.abs(silu) + a) * (np.abs(u) + b)
    return y, size


def weights(rng, out, k, group):
    q = rng.integers(0, 16, (out, k)).astype(np.uint32)
    return q, (0.002 + 0.006 * rng.random((out, k // group))).astype(np.float16)


def close(got, want, size, rel=2e-6):
    assert np.isfinite(got).all()
    assert np.linalg.norm(got - want) <= rel * np.linalg.norm(want), np.linalg.norm(got - want) / np.linalg.norm(want)
    assert (np.abs(got - want) <= 2.0 ** -16 * size).all()


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 31, 32])
@pytest.mark.parametrize("out,k,group", [(16, 128, 32), (5, 128, 128), (33, 384, 64), (2048, 2048, 32), (1000, 1024, 128), (200, 6144, 64)])
def test_gemv(qa, out, k, group, rows):
    rng = np.random.default_rng(out + rows)
    q, d = weights(rng, out, k, group)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    close(gemv(qa, q, d, x, group), *plain(q, d, x))


@pytest.mark.parametrize("rows", [1, 8, 20])
@pytest.mark.parametrize("epi,norm", [(0, True), (1, False), (1, True), (2, False), (2, True)])
def test_epilogues_and_norm(qa, rows, epi, norm):
    rng = np.random.default_rng(rows + 10 * epi)
    out, k, group = 96, 1152, 64
    q, d = weights(rng, out * (2 if epi == 2 else 1), k, group)
    x = (rng.standard_normal((rows, k)) * 3).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32) if norm else None
    y0 = rng.standard_normal((rows, out)).astype(np.float32) if epi == 1 else None
    close(gemv(qa, q, d, x, group, epi, w, y0), *plain(q, d, x, epi, w, y0), rel=8e-6 if epi == 2 else 2e-6)


@pytest.mark.parametrize("rows,k", [(1, 16384), (1, 16512), (2, 24576), (9, 8192), (32, 8320)])
def test_wide_rows(qa, rows, k):
    """More columns than x has room for in LDS: it comes in pieces (sqrt(k / 32 + 128) 2^-24 + 2^-22: 2.1e-6 at 24576)."""
    rng = np.random.default_rng(k)
    q, d = weights(rng, 40, k, 32)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    norm = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    close(gemv(qa, q, d, x, 32, 0, norm), *plain(q, d, x, 0, norm), rel=3e-6)


@pytest.mark.parametrize("rows,epi", [(17, 1), (24, 2), (25, 1), (32, 2)])
def test_two_halves_of_the_rows(qa, rows, epi):
    """More than 16 rows of 2048 columns run as two halves, each with its own x and y."""
    rng = np.random.default_rng(rows)
    out, k, group = 48, 2048, 64
    q, d = weights(rng, out * (2 if epi == 2 else 1), k, group)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    norm = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    y0 = rng.standard_normal((rows, out)).astype(np.float32) if epi == 1 else None
    close(gemv(qa, q, d, x, group, epi, norm, y0), *plain(q, d, x, epi, norm, y0), rel=8e-6 if epi == 2 else 2e-6)


@pytest.mark.parametrize("rows,k,group", [(1, 256, 64), (3, 256, 32), (9, 384, 128), (20, 256, 64), (32, 128, 32)])
def test_vocabulary(qa, rows, k, group):
    """As many rows as the LM head has: workgroups that take several units each, with and without a join."""
    rng = np.random.default_rng(rows)
    q, d = weights(rng, 151936, k, group)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    close(gemv(qa, q, d, x, group), *plain(q, d, x))


@pytest.mark.parametrize("rows,k", [(2, 128), (8, 384)])
def test_many_gated_rows(qa, rows, k):
    rng = np.random.default_rng(k)
    q, d = weights(rng, 2 * 70016, k, 32)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    close(gemv(qa, q, d, x, 32, 2), *plain(q, d, x, 2), rel=8e-6)


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-6, 1e5, 1e30])
def test_magnitudes_of_x(qa, scale):
    """x far outside f16's range; rows of unlike size side by side (each has its own power of two)."""
    rng = np.random.default_rng(4)
    q, d = weights(rng, 64, 512, 32)
    x = rng.standard_normal((4, 512)).astype(np.float32)
    x[1:3] *= np.float32(scale)
    x[3] = 0.0
    got = gemv(qa, q, d, x, 32).astype(np.float64)
    want, size = plain(q, d, x)
    assert (got[3] == 0).all()
    for r in range(3):
        # 2^-149 per value of x where x itself is subnormal, and the result's own subnormal rounding
        tiny = 512 * 2.0 ** -149
        assert np.linalg.norm(got[r] - want[r]) <= 2e-6 * np.linalg.norm(want[r]) + tiny, (r, scale)


def test_norm_of_large_x(qa):
    """Squares are summed in 64 bits: x whose sum of squares passes f32's range, but not its mean."""
    rng = np.random.default_rng(8)
    q, d = weights(rng, 32, 2048, 32)
    x = (rng.standard_normal((3, 2048)) * 3e18).astype(np.float32)
    norm = np.ones(2048, np.float32)
    close(gemv(qa, q, d, x, 32, 0, norm), *plain(q, d, x, 0, norm))


@pytest.mark.parametrize("norm", [False, True])
def test_outliers_in_x(qa, norm):
    """One value 2^20 times the others: the rest keeps its bits."""
    rng = np.random.default_rng(5)
    q, d = weights(rng, 64, 512, 32)
    x = rng.standard_normal((2, 512)).astype(np.float32)
    q[:, 7] = 8                     # weight 0 for the outlier's column
    x[0, 7] = 2.0 ** 20
    w = np.ones(512, np.float32) if norm else None
    got = gemv(qa, q, d, x, 32, 0, w)
    want, size = plain(q, d, x, 0, w)
    # x[0] is split in units of 2^6 (2^20 goes to 2^14); second parts below 2^-14 of a unit are f16 subnormals, off by at
    # most 2^-25 of it: 2^-19 for each x, times the factor of RMSNorm, over all weights
    f = 1 / np.sqrt((x[0].astype(np.float64) ** 2).mean()) if norm else 1.0
    step = 2.0 ** -19 * f * np.linalg.norm(values(q, d))
    assert np.linalg.norm(got[0] - want[0]) <= 2e-6 * np.linalg.norm(want[0]) + step
    close(got[1:], want[1:], size[1:])


def test_not_finite_x(qa):
    """An infinity stays one (NaN where its weight is 0), NaN stays NaN, other rows are untouched."""
    rng = np.random.default_rng(6)
    q, d = weights(rng, 32, 256, 64)
    q[:16, 9], q[16:31, 9], q[31, 9] = 12, 3, 8
    x = rng.standard_normal((4, 256)).astype(np.float32)
    x[0, 9], x[1, 9], x[2, 9] = np.inf, -np.inf, np.nan
    got = gemv(qa, q, d, x, 64)
    assert (got[0, :16] == np.inf).all() and (got[0, 16:31] == -np.inf).all() and np.isnan(got[0, 31])
    assert (got[1, :16] == -np.inf).all() and (got[1, 16:31] == np.inf).all() and np.isnan(got[1, 31])
    assert np.isnan(got[2]).all()
    want, size = plain(q, d, x[3:])
    close(got[3:], want, size)


def test_pack_then_multiply(qa):
    rng = np.random.default_rng(7)
    out, k, group = 80, 512, 32
    w = (rng.standard_normal((out, k)) * 0.02).astype(np.float32)
    x = rng.standard_normal((1, k)).astype(np.float32)
    src, dx = qa.DeviceArray.from_numpy(w), qa.DeviceArray.from_numpy(x)
    dw, ds = qa.DeviceArray((qa.lib.qa_q4_weight_bytes(out, k),), np.uint8), qa.DeviceArray((qa.lib.qa_q4_scale_count(out, k, group),), np.uint16)
    y = qa.DeviceArray((1, out))
    qa.check(qa.lib.qa_pack_q4(src.ptr, out, k, group, dw.ptr, ds.ptr, None))
    qa.check(qa.lib.qa_gemv_q4(dw.ptr, ds.ptr, group, out, k, dx.ptr, 1, y.ptr, 0, None, 1e-6, None))
    qa.synchronize()
    q, d = quantise(w, group)
    close(y.numpy(), *plain(q, d, x))


@pytest.mark.parametrize("rows,k,epi", [(17, 2048, 1), (28, 2048, 2), (32, 512, 0), (13, 2048, 2), (32, 2176, 0)])
def test_many_tiles_and_rows(qa, rows, k, epi):
    """More tiles than workgroups run at a time, and up to 32 rows: x once in LDS, in two parts, or with every tile."""
    rng = np.random.default_rng(rows)
    out, group = 8208, 128
    q, d = weights(rng, out * (2 if epi == 2 else 1), k, group)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    norm = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    y0 = rng.standard_normal((rows, out)).astype(np.float32) if epi == 1 else None
    close(gemv(qa, q, d, x, group, epi, norm, y0), *plain(q, d, x, epi, norm, y0), rel=8e-6 if epi == 2 else 2e-6)


@pytest.mark.parametrize("rows", [6, 14, 30])
@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-6, 1e5, 1e30])
def test_magnitudes_of_x_in_more_rows(qa, rows, scale):
    rng = np.random.default_rng(rows)
    q, d = weights(rng, 64, 2304, 32)
    x = rng.standard_normal((rows, 2304)).astype(np.float32)
    x[1::3] *= np.float32(scale)
    x[3] = 0.0
    got = gemv(qa, q, d, x, 32).astype(np.float64)
    want, size = plain(q, d, x)
    assert (got[3] == 0).all()
    for r in range(rows):
        tiny = 2304 * 2.0 ** -149
        assert np.linalg.norm(got[r] - want[r]) <= 2e-6 * np.linalg.norm(want[r]) + tiny, (r, scale)


@pytest.mark.parametrize("rows", [5, 12, 32])
@pytest.mark.parametrize("norm", [False, True])
def test_columns_of_unlike_size(qa, rows, norm):
    """Columns that grow and shrink by 2^40 along a row: whatever is split first, the large ones keep their bits."""
    rng = np.random.default_rng(rows)
    k = 128 * 41
    q, d = weights(rng, 48, k, 64)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    up = np.exp2(np.arange(k) // 128 - 20).astype(np.float32)
    x[0] *= up
    x[1] *= up[::-1]
    x[2] *= rng.permutation(up)
    x[3, :128 * 40] = 0.0
    w = np.ones(k, np.float32) if norm else None
    close(gemv(qa, q, d, x, 64, 0, w), *plain(q, d, x, 0, w))


@pytest.mark.parametrize("rows", [7, 15, 32])
@pytest.mark.parametrize("norm", [False, True])
def test_not_finite_x_in_more_rows(qa, rows, norm):
    rng = np.random.default_rng(6)
    q, d = weights(rng, 32, 2304, 64)
    q[:16, 2009], q[16:31, 2009], q[31, 2009] = 12, 3, 8
    x = rng.standard_normal((rows, 2304)).astype(np.float32)
    x[0, 2009], x[1, 2009], x[2, 2009], x[4, 2009] = np.inf, -np.inf, np.nan, 3e38
    w = np.ones(2304, np.float32) if norm else None
    got = gemv(qa, q, d, x, 64, 0, w)
    if norm:
        assert np.isnan(got[:3]).all()                            # inf times its row's factor 0
    else:
        assert (got[0, :16] == np.inf).all() and (got[0, 16:31] == -np.inf).all() and np.isnan(got[0, 31])
        assert (got[1, :16] == -np.inf).all() and (got[1, 16:31] == np.inf).all() and np.isnan(got[1, 31])
        assert np.isnan(got[2]).all()
    rest = [3] + list(range(5, rows))
    want, size = plain(q, d, x[rest], 0, w)
    close(got[rest], want, size)
    assert np.isfinite(got[4]).all()


@pytest.mark.parametrize("rows", [3, 7, 20])
def test_norm_of_large_x_in_more_rows(qa, rows):
    """The sum of squares, and x times its weights, pass f32's range before the factor brings them back."""
    rng = np.random.default_rng(8)
    q, d = weights(rng, 32, 2304, 32)
    x = (rng.standard_normal((rows, 2304)) * 3e18).astype(np.float32)
    norm = np.full(2304, 1e18, np.float32)
    close(gemv(qa, q, d, x, 32, 0, norm), *plain(q, d, x, 0, norm))


@pytest.mark.parametrize("epi,norm", [(0, False), (0, True), (1, True), (2, True)])
@pytest.mark.parametrize("out,k,group", [(40, 1920, 32), (4096 + 16, 2048, 64), (8208, 512, 128), (16, 128 * 65, 32), (12304, 256, 32)])
def test_single_row(qa, out, k, group, epi, norm):
    """One token: column blocks that do not come out even over the waves, more than 64 of them, several tiles per workgroup."""
    rng = np.random.default_rng(k + epi)
    out = -(-out // 16) * 16 if epi == 2 else out
    q, d = weights(rng, out * (2 if epi == 2 else 1), k, group)
    x = (rng.standard_normal((1, k)) * 3).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32) if norm else None
    y0 = rng.standard_normal((1, out)).astype(np.float32) if epi == 1 else None
    close(gemv(qa, q, d, x, group, epi, w, y0), *plain(q, d, x, epi, w, y0), rel=8e-6 if epi == 2 else 2e-6)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("kind", ["up", "down", "mixed", "last", "tiny", "huge", "zero"])
def test_single_row_of_unlike_columns(qa, kind, norm):
    rng = np.random.default_rng(11)
    k = 128 * 83
    q, d = weights(rng, 48, k, 64)
    x = rng.standard_normal((1, k)).astype(np.float32)
    up = np.exp2(np.arange(k) // 256 - 20).astype(np.float32)
    if kind == "up":
        x *= up
    elif kind == "down":
        x *= up[::-1]
    elif kind == "mixed":
        x *= rng.permutation(up)
    elif kind == "last":
        x[:, :-1] = 0.0
    elif kind == "tiny":
        x *= np.float32(1e-30)
    elif kind == "huge":
        x *= np.float32(1e30 if not norm else 1e18)
    else:
        x[:] = 0.0
    w = np.ones(k, np.float32) if norm else None
    got = gemv(qa, q, d, x, 64, 0, w)
    want, size = plain(q, d, x, 0, w)
    if kind == "zero":
        assert (got == 0).all()
    else:
        assert np.isfinite(got).all()
        assert np.linalg.norm(got - want) <= 3e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("at", [0, 1029, 2303, 8400])
def test_single_row_not_finite(qa, value, at):
    rng = np.random.default_rng(at)
    k = 128 * 66
    q, d = weights(rng, 32, k, 64)
    q[:16, at], q[16:31, at], q[31, at] = 12, 3, 8
    x = rng.standard_normal((1, k)).astype(np.float32)
    x[0, at] = value
    got = gemv(qa, q, d, x, 64)[0]
    if np.isnan(value):
        assert np.isnan(got).all()
    else:
        assert (got[:16] == value).all() and (got[16:31] == -value).all() and np.isnan(got[31])
