"""A paged cache of 8 bits: rows quantised as they are appended, read back, attended and moved, against plain 64-bit statements.

Tolerances.  Attention reads the stored numbers, int8 * scale: products and sums are f32, so the bounds are those of the other
cache types (a score sqrt(128) 2^-24 |s| off, a probability as much, sums of L rows sqrt(L) 2^-25): 5e-6 in the 2-norm, 2^-16 of
the largest |v| for one value.  Appended rows: an f32 row is within 2^-20 of its largest value (six roundings), so its scale
is within 2^-20 + 2^-24 of itself, and a stored value is off by half a step and what the row is off by, 127 2^-20 of a step;
it is the nearest integer of the exact row but where that lies within 2^-12 of a border (127 (2^-20 + 2^-20 + 2^-24) < 2^-12)."""
import ctypes as C

import numpy as np
import pytest

import candidates_ref as cand
import paged_ref as ref

pytestmark = pytest.mark.gpu

REL, MAX = 5e-6, 2.0 ** -16


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


def close(got, want, vmax):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert np.isfinite(got).all()
    rel = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    assert rel <= REL and np.abs(got - want).max() <= MAX * vmax, (rel, np.abs(got - want).max() / vmax)


def case(qa, seed, past, news, page, kv_heads=8, group=2, layers=2, layer=1, n_rows=None, fill=0.0, workspace=None, holes=(),
         change=None, **bounds):
    rng = np.random.default_rng(seed)
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], page)
    for s, j, to in holes:
        tables[s, j] = to
    pool = cand.Pool(qa, "q8", layers, pages, kv_heads, page, rng)
    if change:
        change(pool, tables)
    heads = kv_heads * group
    b = ref.Batch(qa, tables, past, news, n_rows=n_rows, **bounds)
    q = rng.standard_normal((b.rows, heads * 128)).astype(np.float32)
    print(f"q8 attention past={past} news={news} page={page} kv_heads={kv_heads} group={group} holes={len(holes)}", flush=True)
    got = cand.run_attention(qa, q, pool, layer, b, heads, fill=fill, workspace=workspace)
    want = ref.attention(q, pool.values, layer, tables, page, b.past, b.start, heads, out=np.full((b.rows, heads, 128), fill))
    return got, want, pool


@pytest.mark.parametrize("past,news,page", [
    ([0], [1], 16), ([15], [1], 16), ([16], [1], 16), ([31], [1], 16), ([156], [1], 16), ([31, 32, 33, 0], [1, 1, 1, 1], 32),
    ([63, 200, 5], [1, 2, 4], 64), ([1000], [1], 128), ([700], [3], 256), ([3930], [1], 16), ([0], [5], 16), ([0], [33], 16),
    ([0], [64], 32), ([10], [65], 16), ([100, 0, 7], [40, 0, 129], 64), ([5, 300, 0, 77, 0], [1, 130, 0, 9, 17], 16),
    ([511], [257], 256), ([0, 0, 0], [0, 3, 0], 16), ([3000], [300], 32), ([2500, 40], [600, 1], 16),
])
def test_attention(qa, past, news, page):
    got, want, pool = case(qa, 1 + len(past) * 7 + past[0], past, news, page)
    close(got, want, np.abs(pool.values).max())


@pytest.mark.parametrize("kv_heads,group,news", [(1, 1, 20), (2, 3, 1), (2, 3, 37), (4, 8, 1), (3, 16, 1), (1, 16, 30), (8, 1, 8), (5, 5, 3),
                                                 (8, 4, 2), (8, 4, 3), (8, 1, 9), (8, 2, 8)])
def test_head_layouts(qa, kv_heads, group, news):
    got, want, pool = case(qa, 31 + kv_heads, [50, 9], [news, 1], 32, kv_heads=kv_heads, group=group)
    close(got, want, np.abs(pool.values).max())


def test_rows_of_no_sequence_and_no_bounds(qa):
    got, want, pool = case(qa, 5, [40, 0, 600], [1, 70, 2], 16, n_rows=80, fill=7.25, max_tokens=0, max_len=0)
    close(got[:73], want[:73], np.abs(pool.values).max())
    assert (got[73:] == 7.25).all()


@pytest.mark.parametrize("past,news,holes", [
    ([60], [1], [(0, 1, -1)]), ([60], [40], [(0, 0, -1), (0, 2, -5)]), ([20], [20], [(0, 0, -1), (0, 1, -1), (0, 2, -1)]),
    ([40, 3], [1, 1], [(1, 0, 2 ** 31 - 1)]), ([500], [70], [(0, j, -1) for j in range(0, 30)]), ([2600], [300], [(0, j, -1) for j in range(3, 90, 7)]),
])
def test_positions_without_a_page(qa, past, news, holes):
    got, want, pool = case(qa, 13, past, news, 16, holes=holes, fill=5.0)
    close(got, want, np.abs(pool.values).max())


@pytest.mark.parametrize("past,news", [([37], [1]), ([37], [30]), ([90, 13], [1, 70]), ([2600], [300])])
def test_what_masked_places_hold_does_not_matter(qa, past, news):
    """Scales of free pages, of the rest of the last page and of later tokens are NaN or infinite: earlier tokens do not see them."""
    def change(pool, tables):
        held = np.zeros(pool.layout.n_streams, bool)
        change.clean = cand.Pool(qa, "q8", 1, 1, 1, 16)
        change.clean.ints, change.clean.scales = pool.ints.copy(), pool.scales.copy()
        for s, (p, n) in enumerate(zip(past, news)):
            for j in range(p + n):
                held[tables[s, j // 16]] = True
            last = p + n - 1
            if (last + 1) % 16:
                pool.scales[:, :, tables[s, last // 16], :, last % 16 + 1:] = np.nan
            pool.scales[:, 1, tables[s, last // 16], :, last % 16] = np.nan      # the last token's own row
        pool.scales[:, :, ~held] = np.inf
        pool.ints[:, :, ~held] = -128
    got, want, pool = case(qa, 3, past, news, 16, layers=1, layer=0, change=change)
    first = 0
    for n in news:
        assert np.isnan(got[first + n - 1]).all()
        if n > 1:
            close(got[first:first + n - 1], want[first:first + n - 1], np.abs(change.clean.values).max())
        first += n


@pytest.mark.parametrize("past,news", [([900], [1]), ([300], [40]), ([2600], [300])])
@pytest.mark.parametrize("spread", [1, 24, 60, 110])
def test_scales_of_very_different_size(qa, past, news, spread):
    """V rows whose scales lie up to 2^spread apart, small ones first and last; the error counts against the sizes that are met."""
    def change(pool, tables):
        rng = np.random.default_rng(spread)
        pool.scales[:, 1] *= np.exp2(rng.integers(-spread // 2, spread // 2 + 1, pool.scales[:, 1].shape)).astype(np.float32)
        pool.scales[:, 0, ::3] *= np.float32(0.25)
    got, want, pool = case(qa, 9, past, news, 16, layers=1, layer=0, kv_heads=2, change=change)
    close(got, want, np.abs(pool.values[:, 1]).max())


def test_rows_of_zeros(qa):
    """Scales of 0, for all keys and for some: values are zeros, and keys of zeros still have their weight."""
    def zeros(pool, tables):
        pool.scales[:, 1] = 0
    got, *_ = case(qa, 2, [200], [1], 16, change=zeros)
    assert (got == 0).all()

    def some(pool, tables):
        pool.scales[:, 1, ::2] = 0
        pool.scales[:, 0, 1::2] = 0
    got, want, pool = case(qa, 2, [200, 17], [1, 30], 16, change=some)
    close(got, want, np.abs(pool.values).max())


def test_less_workspace(qa):
    a, want, pool = case(qa, 4, [3900, 20], [1, 1], 16)
    b, *_ = case(qa, 4, [3900, 20], [1, 1], 16, workspace=0)
    close(a, want, np.abs(pool.values).max())
    close(b, want, np.abs(pool.values).max())


def appended(qa, cache, past, news, page, kv_heads=8, group=2, seed=6, qkv=None, depth=None, spare_rows=0, holes=()):
    """(q, pool, read k, read v, the batch, its tables and inputs) after an append into a pool of old values."""
    rng = np.random.default_rng(seed)
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], page)
    for s, j, to in holes:
        tables[s, j] = to
    pool = cand.Pool(qa, cache, 2, pages, kv_heads, page, rng)
    heads = kv_heads * group
    b = ref.Batch(qa, tables, past, news, n_rows=sum(news) + spare_rows)
    if qkv is None:
        qkv = rng.standard_normal((b.rows, (heads + 2 * kv_heads) * 128)).astype(np.float32)
    wq, wk = (1 + 0.1 * rng.standard_normal(128)).astype(np.float32), (1 + 0.1 * rng.standard_normal(128)).astype(np.float32)
    d = [qa.DeviceArray.from_numpy(a) for a in (qkv, wq, wk)]
    d_pool = pool.upload()
    q = qa.DeviceArray.from_numpy(np.full((b.rows, heads * 128), 9.0, np.float32))
    if depth is None:
        qa.check(qa.lib.qa_paged_append(d[0].ptr, d[1].ptr, d[2].ptr, q.ptr, d_pool.ptr, C.byref(pool.layout), 1, b.ref, heads, 1e6, 1e-6, None))
    else:
        d_depth = qa.DeviceArray.from_numpy(np.asarray(depth, np.int32))
        qa.check(qa.lib.qa_paged_tree_append(d[0].ptr, d[1].ptr, d[2].ptr, q.ptr, d_pool.ptr, C.byref(pool.layout), 1, b.ref, d_depth.ptr, heads,
                                             1e6, 1e-6, None))
    out = {}
    for name, kind, dtype in (("f32", qa.QA_CACHE_F32, np.float32), ("f16", qa.QA_CACHE_F16, np.float16)):
        k, v = (qa.DeviceArray.from_numpy(np.full((b.rows, kv_heads, 128), 5.0, dtype)) for _ in range(2))
        qa.check(qa.lib.qa_paged_read(d_pool.ptr, C.byref(pool.layout), 1, b.ref, k.ptr, v.ptr, kind, None))
        qa.synchronize()
        out[name] = k.numpy(), v.numpy()
    return q.numpy().reshape(b.rows, heads, 128), pool, pool.take(d_pool.numpy()), out, b, tables, qkv, wq, wk


@pytest.mark.parametrize("past,news,page", [([0], [1], 16), ([15], [2], 16), ([156, 0, 700], [1, 40, 3], 32), ([3900], [9], 64), ([0], [1100], 256)])
@pytest.mark.parametrize("kv_heads,group", [(8, 2), (3, 1)])
def test_append_and_read(qa, past, news, page, kv_heads, group):
    q, old, pool, out, b, tables, qkv, wq, wk = appended(qa, "q8", past, news, page, kv_heads, group)
    heads = kv_heads * group
    x = qkv.reshape(b.rows, -1, 128)
    seen = np.zeros(pool.scales.shape, bool)
    for s, (p, n) in enumerate(zip(past, news)):
        for t in range(n):
            r, pos = b.start[s] + t, p + t
            pg, sl = tables[s, pos // page], pos % page
            want_q = ref.rope_norm(x[r, :heads], wq, pos)
            assert np.abs(q[r] - want_q).max() <= 2.0 ** -20 * np.abs(want_q).max()
            want = ref.rope_norm(x[r, heads:heads + kv_heads], wk, pos), x[r, heads + kv_heads:].astype(np.float64)
            for kv in (0, 1):
                seen[1, kv, pg, :, sl] = True
                scale, ints = pool.scales[1, kv, pg, :, sl].astype(np.float64), pool.ints[1, kv, pg, :, sl].astype(np.float64)
                exact = np.abs(want[kv]).max(-1) / 127
                assert np.abs(scale / exact - 1).max() <= 2.0 ** -20 + 2.0 ** -24 + (kv == 0) * 2.0 ** -20
                steps = want[kv] / exact[:, None]
                assert np.abs(ints - steps).max() <= 0.5 + 2.0 ** -12
                if kv == 1:      # v is stored as it came: the very integers
                    wi, ws = cand.quantise(x[r, heads + kv_heads:])
                    np.testing.assert_array_equal(pool.ints[1, 1, pg, :, sl], wi)
                    np.testing.assert_array_equal(pool.scales[1, 1, pg, :, sl], ws)
                stands = pool.ints[1, kv, pg, :, sl].astype(np.float32) * pool.scales[1, kv, pg, :, sl][:, None]
                np.testing.assert_array_equal(out["f32"][kv][r], stands)
                np.testing.assert_array_equal(out["f16"][kv][r], stands.astype(np.float16))
    # every other row is what it was
    np.testing.assert_array_equal(pool.ints[~seen], old.ints[~seen])
    np.testing.assert_array_equal(pool.scales[~seen], old.scales[~seen])


def test_append_of_rows_that_are_not_ordinary(qa):
    """Zeros, the smallest numbers, the largest, infinities and NaN in V."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((6, 4, 128)).astype(np.float32)
    tiny = np.float32(1e-45)
    x[0, 3] = 0
    x[1, 3] = tiny * rng.integers(-200, 201, 128)
    x[2, 3] *= np.float32(1e-36)
    x[3, 3] *= np.float32(6e37)
    x[4, 3, 77] = np.inf
    x[5, 3, 3] = np.nan
    q, old, pool, out, b, tables, *_ = appended(qa, "q8", [10], [6], 16, 1, 2, qkv=x.reshape(6, -1))
    for r in range(6):
        pg, sl = tables[0, (10 + r) // 16], (10 + r) % 16
        wi, ws = cand.quantise(x[r, 3])
        np.testing.assert_array_equal(pool.scales[1, 1, pg, 0, sl], ws)
        if r < 4:
            np.testing.assert_array_equal(pool.ints[1, 1, pg, 0, sl], wi)
            assert np.isfinite(out["f32"][1][r]).all()
        else:
            assert np.isnan(out["f32"][1][r]).all() and np.isnan(out["f16"][1][r]).all()


@pytest.mark.parametrize("cache", cand.CACHES)
def test_read_of_every_cache(qa, cache):
    """The values of any cache as f32 and f16; rows on no page are zeros, rows of no sequence stay."""
    q, old, pool, out, b, tables, *_ = appended(qa, cache, [5, 40], [30, 2], 16, spare_rows=3, holes=[(0, 1, -1)])
    for r in range(35):
        s, pos = (0, 5 + r) if r < 30 else (1, 40 + r - 30)
        for kv in (0, 1):
            if r >= 32:
                assert (out["f32"][kv][r] == 5).all() and (out["f16"][kv][r] == 5).all()
                continue
            pg = tables[s, pos // 16]
            want = pool.values[1, kv, pg, :, pos % 16].astype(np.float32) if pg >= 0 else np.zeros((8, 128), np.float32)
            np.testing.assert_array_equal(out["f32"][kv][r], want)
            np.testing.assert_array_equal(out["f16"][kv][r], want.astype(np.float16))


def test_read_of_one_side(qa):
    rng = np.random.default_rng(1)
    tables, pages = ref.tables_of(rng, [20], 16)
    pool = cand.Pool(qa, "q8", 1, pages, 2, 16, rng)
    b = ref.Batch(qa, tables, [0], [20])
    d_pool, v = pool.upload(), qa.DeviceArray((20, 2, 128))
    qa.check(qa.lib.qa_paged_read(d_pool.ptr, C.byref(pool.layout), 0, b.ref, None, v.ptr, qa.QA_CACHE_F32, None))
    qa.synchronize()
    for r in range(20):
        np.testing.assert_array_equal(v.numpy()[r], pool.values[0, 1, tables[0, r // 16], :, r % 16].astype(np.float32))


def test_pages_of_8_bits_are_given_copied_and_moved(qa):
    """qa_kv_cache_alloc, extend with copies, copy and compact move a page's values and scales."""
    rng = np.random.default_rng(2)
    pool = cand.Pool(qa, "q8", 2, 9, 3, 16, rng)
    lay = C.byref(pool.layout)
    tables = np.array([[7, 2, -1], [7, 2, -1]], np.int32)
    refs = np.bincount(tables[tables >= 0], minlength=9).astype(np.int32)
    d_pool, d_t, d_r = pool.upload(), qa.DeviceArray.from_numpy(tables), qa.DeviceArray.from_numpy(refs)
    ints = [qa.DeviceArray.from_numpy(np.array(v, np.int32)) for v in ([1], [20], [1])]
    missing, live = qa.DeviceArray((1,), np.int32), qa.DeviceArray((1,), np.int32)
    need = qa.lib.qa_pages_workspace_bytes(lay)
    ws = qa.DeviceArray((need,), np.uint8)
    qa.check(qa.lib.qa_pages_extend(d_pool.ptr, lay, d_r.ptr, d_t.ptr, 2, 3, ints[0].ptr, ints[1].ptr, ints[2].ptr, 1, missing.ptr, ws.ptr, need, None))
    src, dst = (qa.DeviceArray.from_numpy(np.array(v, np.int32)) for v in ([7], [5]))
    qa.check(qa.lib.qa_pages_copy(d_pool.ptr, lay, src.ptr, dst.ptr, 1, None))
    qa.synchronize()
    got = pool.take(d_pool.numpy())
    assert d_t.numpy().tolist() == [[7, 2, -1], [7, 0, -1]]
    for to, source in ((0, 2), (5, 7)):
        np.testing.assert_array_equal(got.ints[:, :, to], pool.ints[:, :, source])
        np.testing.assert_array_equal(got.scales[:, :, to], pool.scales[:, :, source])
    for same in (1, 2, 3, 4, 6, 7, 8):
        np.testing.assert_array_equal(got.ints[:, :, same], pool.ints[:, :, same])
    qa.check(qa.lib.qa_pages_compact(d_pool.ptr, lay, d_r.ptr, d_t.ptr, 2, 3, d_r.ptr, d_t.ptr, live.ptr, ws.ptr, need, None))
    qa.synchronize()
    last = pool.take(d_pool.numpy())
    assert int(live.numpy()[0]) == 3 and d_t.numpy().tolist() == [[1, 2, -1], [1, 0, -1]]
    np.testing.assert_array_equal(last.ints[:, :, 1], pool.ints[:, :, 7])
    np.testing.assert_array_equal(last.scales[:, :, 1], pool.scales[:, :, 7])
    p = C.c_void_p()
    qa.check(qa.lib.qa_kv_cache_alloc(lay, C.byref(p)))
    qa.check(qa.lib.qa_kv_cache_free(p))
