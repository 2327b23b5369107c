"""Append and attention over a K/V cache in pages, against plain 64-bit statements.

Tolerances.  Attention has f32 products and sums: a score is off by about sqrt(128) 2^-24 |s| (sums of 128 products, |s| < 4
for unit rows: 3e-6 at most), a probability by the same relative amount, and the sum of L weighted rows adds sqrt(L) 2^-25
(2e-6 at L = 4096); the errors of different keys are independent, so the result's relative 2-norm error stays below 5e-6, and
a single value below 2^-16 = 1.5e-5 of the largest |v| that it averages.  Appended rows: q within 2^-20 of its row's largest
value (norm, rotation: six f32 roundings of at most 2^-24 each), cached rows half a step of the cache's type more."""
import ctypes as C

import numpy as np
import pytest

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


def case(qa, seed, past, news, page, f16, kv_heads=8, group=2, layers=2, layer=1, bounds=True, n_rows=None, fill=0.0,
         workspace=None, scale=ref.SCALE, q_scale=1.0, holes=()):
    rng = np.random.default_rng(seed)
    tables, pages = ref.tables_of(rng, [max(p, 0) + n for p, n in zip(past, news)], page)
    for s, j, to in holes:
        tables[s, j] = to(pages) if callable(to) else to
    pool = ref.pool_of(rng, layers, pages, kv_heads, page, f16)
    heads = kv_heads * group
    kw = {} if bounds else dict(max_tokens=0, max_len=0)
    b = ref.Batch(qa, tables, past, news, n_rows=n_rows, **kw)
    q = (rng.standard_normal((b.rows, heads * 128)) * q_scale).astype(np.float32)
    print(f"attention past={past} news={news} page={page} f16={f16} kv_heads={kv_heads} group={group} holes={len(holes)}", flush=True)
    got = ref.run_attention(qa, q, pool, layer, b, page, heads, scale=scale, fill=fill, workspace=workspace)
    want = ref.attention(q, pool, layer, tables, page, b.past, b.start, heads, scale=scale,
                         out=np.full((b.rows, heads, 128), fill))
    return got, want, pool, q, tables, b


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past,news,page", [
    ([0], [1], 16), ([15], [1], 16), ([16], [1], 16), ([156], [1], 16), ([31, 32, 33, 0], [1, 1, 1, 1], 32),
    ([63, 200, 5], [1, 2, 4], 64), ([1000], [1], 128), ([700], [3], 256), ([3930], [1], 16),
    ([0], [5], 16), ([0], [33], 16), ([0], [64], 32), ([10], [65], 16), ([100, 0, 7], [40, 0, 129], 64),
    ([5, 300, 0, 77, 0], [1, 130, 0, 9, 17], 16), ([511], [257], 256), ([0, 0, 0], [0, 3, 0], 16),
])
def test_attention(qa, f16, past, news, page):
    got, want, pool, *_ = case(qa, 1 + len(past) * 7 + past[0], past, news, page, f16)
    close(got, want, np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("kv_heads,group,news", [(1, 1, 20), (2, 3, 1), (2, 3, 37), (4, 8, 1), (3, 16, 1), (1, 16, 30), (8, 1, 8), (5, 5, 3),
                                                 (8, 4, 2), (8, 4, 3), (8, 1, 9), (8, 2, 8), (8, 2, 9)])
def test_head_layouts(qa, f16, kv_heads, group, news):
    got, want, pool, *_ = case(qa, 31 + kv_heads, [50, 9], [news, 1], 32, f16, kv_heads=kv_heads, group=group)
    close(got, want, np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
def test_bounds_of_the_host_are_optional(qa, f16):
    """Without max_tokens and max_len the device's numbers decide; rows behind the last sequence keep what they held."""
    past, news = [40, 0, 600], [1, 70, 2]
    got, want, pool, *_ = case(qa, 5, past, news, 16, f16, bounds=False, n_rows=80, fill=7.25)
    close(got[:73], want[:73], np.abs(pool.astype(np.float64)).max())
    assert (got[73:] == 7.25).all()


@pytest.mark.parametrize("f16", [True, False])
def test_rows_before_the_first_sequence_and_idle_ones(qa, f16):
    rng = np.random.default_rng(8)
    tables, pages = ref.tables_of(rng, [30, 30, 30], 16)
    pool = ref.pool_of(rng, 1, pages, 8, 16, f16)
    b = ref.Batch(qa, tables, [20, 20, 20], [1, 0, 2], n_rows=9)
    b.start = np.array([3, 4, 4, 6], np.int32)
    b.d[2].upload(b.start)
    q = rng.standard_normal((9, 2048)).astype(np.float32)
    got = ref.run_attention(qa, q, pool, 0, b, 16, 16, fill=-3.0)
    want = ref.attention(q, pool, 0, tables, 16, b.past, b.start, 16)
    close(got[3:6], want[3:6], np.abs(pool.astype(np.float64)).max())
    assert (got[:3] == -3.0).all() and (got[6:] == -3.0).all()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("news", [1, 40])
def test_many_sequences(qa, f16, news):
    """More than one wave's worth of sequences, most of them short, some idle."""
    rng = np.random.default_rng(news)
    n = 150
    past = rng.integers(0, 60, n).tolist()
    tokens = [int(rng.integers(0, 3)) if i % 9 else news for i in range(n)]
    got, want, pool, *_ = case(qa, 77, past, tokens, 16, f16, kv_heads=2)
    close(got, want, np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past,news,holes", [
    ([60], [1], [(0, 1, -1)]), ([60], [40], [(0, 0, -1), (0, 2, -5)]), ([100], [1], [(0, 0, lambda n: n), (0, 6, 2 ** 31 - 1)]),
    ([20], [20], [(0, 0, -1), (0, 1, -1), (0, 2, -1)]), ([40, 3], [1, 1], [(1, 0, -1)]), ([0], [50], [(0, 0, -1)]),
    ([500], [70], [(0, j, -1) for j in range(0, 30)]),
])
def test_positions_without_a_page(qa, f16, past, news, holes):
    """Page numbers outside the cache are no pages; a token that sees no position gets zeros."""
    got, want, pool, q, tables, b = case(qa, 13, past, news, 16, f16, holes=holes, fill=5.0)
    close(got, want, np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past,news", [([37], [1]), ([37], [30]), ([90, 13], [1, 70])])
def test_what_masked_places_hold_does_not_matter(qa, f16, past, news):
    """Free pages, the rest of the last page and later tokens' V are NaN or infinite: earlier tokens do not see it."""
    rng = np.random.default_rng(3)
    page = 16
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], page)
    pool = ref.pool_of(rng, 1, pages, 8, page, f16)
    clean = pool.copy()
    held = np.zeros(pages, bool)
    for s, (p, n) in enumerate(zip(past, news)):
        for j in range(p + n):
            held[tables[s, j // page]] = True
        last = p + n - 1
        if (last + 1) % page:
            pool[:, :, tables[s, last // page], :, last % page + 1:] = np.nan
        # the last token's own row: only it may become NaN
        pool[:, 1, tables[s, last // page], :, last % page, ::3] = np.inf
        pool[:, 0, tables[s, last // page], :, last % page, 5] = np.nan
    pool[:, :, ~held] = np.inf
    b = ref.Batch(qa, tables, past, news)
    q = rng.standard_normal((b.rows, 2048)).astype(np.float32)
    got = ref.run_attention(qa, q, pool, 0, b, page, 16)
    want = ref.attention(q, clean, 0, tables, page, b.past, b.start, 16)
    last = b.start[1:] - 1
    others = np.setdiff1d(np.arange(b.rows), last)
    assert np.isnan(got[last]).all()
    if len(others):
        close(got[others], want[others], np.abs(clean.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("news", [1, 20])
def test_infinities_follow_the_formula(qa, f16, news):
    rng = np.random.default_rng(21)
    tables, pages = ref.tables_of(rng, [80 + news], 16)
    pool = ref.pool_of(rng, 1, pages, 8, 16, f16)
    pool[0, 1, tables[0, 1], 0, 3, 10] = np.inf       # a visible V: that value of head 0's rows is inf
    pool[0, 1, tables[0, 2], 1, 4, 11] = -np.inf
    pool[0, 0, tables[0, 3], 2, 5, :] = 0.0
    pool[0, 0, tables[0, 3], 2, 5, 0] = -np.inf       # with q > 0 there: score -inf, no weight
    b = ref.Batch(qa, tables, [80], [news])
    q = np.abs(rng.standard_normal((b.rows, 2048))).astype(np.float32)
    q.reshape(-1, 16, 128)[:, 14] = 0.0               # a zero row: every visible key alike
    got = ref.run_attention(qa, q, pool, 0, b, 16, 16)
    want = ref.attention(q, pool, 0, tables, 16, b.past, b.start, 16)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert (got[:, :2, 10] == np.inf).all() and (got[:, 2:4, 11] == -np.inf).all() and np.isfinite(got[:, 4:]).all()
    fine = np.isfinite(want)
    close(got[fine], want[fine], 6.0)


@pytest.mark.parametrize("f16", [True, False])
def test_all_visible_scores_minus_infinity(qa, f16):
    """softmax of nothing but -inf is NaN, not the zeros of a token that sees no position."""
    rng = np.random.default_rng(2)
    tables, pages = ref.tables_of(rng, [40], 16)
    pool = ref.pool_of(rng, 1, pages, 8, 16, f16)
    pool[0, 0] = 0.0
    pool[0, 0, ..., 0] = -np.inf
    b = ref.Batch(qa, tables, [37], [3])
    q = np.ones((3, 2048), np.float32)
    assert np.isnan(ref.run_attention(qa, q, pool, 0, b, 16, 16)).all()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("q_scale,scale", [(1e-30, 1e28), (1e4, 1e-5), (300.0, 3e-4), (1e30, 1e-31), (3.0, 1.0)])
def test_magnitudes_of_q(qa, f16, q_scale, scale):
    """q far outside f16's range, small and large; scores of a sharp softmax (|s| up to 150) are off by up to 2^-24 * 128
    of the sum of |q k|, so the last pair is held to 64 times the bar."""
    got, want, pool, *_ = case(qa, 9, [70], [9], 16, f16, q_scale=q_scale, scale=scale)
    vmax = np.abs(pool.astype(np.float64)).max()
    close(want + (got - want) / (64 if scale == 1.0 else 1), want, vmax)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past,news", [([3000], [1]), ([1500, 20], [70, 1])])
def test_any_workspace(qa, f16, past, news):
    """Without a workspace, with a part of it, with all: the same result to the tolerance; with the same one the same bits."""
    args = (qa, 4, past, news, 32, f16)
    full, want, pool, *_ = case(*args)
    vmax = np.abs(pool.astype(np.float64)).max()
    again = case(*args)[0]
    np.testing.assert_array_equal(full.view(np.uint32), again.view(np.uint32))
    rows = sum(news)
    for size in (0, rows * 16 * 130 * 4 * 2 - 16, rows * 16 * 130 * 4 * 3):
        close(case(*args, workspace=size)[0], want, vmax)


def test_growing_maximum_and_long_tail(qa):
    """Scores that rise along the keys move the reference maximum many times; one key holds nearly all the weight."""
    for f16 in (True, False):
        rng = np.random.default_rng(6)
        tables, pages = ref.tables_of(rng, [900], 64)
        pool = ref.pool_of(rng, 1, pages, 8, 64, f16)
        u = rng.standard_normal(128)
        u /= np.linalg.norm(u)
        for j in range(900):
            pool[0, 0, tables[0, j // 64], :, j % 64] = (u * (0.5 * j)).astype(pool.dtype)
        b = ref.Batch(qa, tables, [890], [10])
        q = np.tile((u * 1.0).astype(np.float32), (10, 16))
        got = ref.run_attention(qa, q, pool, 0, b, 64, 16, scale=1.0)
        want = ref.attention(q, pool, 0, tables, 64, b.past, b.start, 16, scale=1.0)
        # |s| up to 450: scores off by up to 450 * 128 * 2^-24 / 8 (eight products are summed per lane) = 4e-4
        assert np.abs(got - want).max() <= 4e-4 * 2 * 6


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("news", [[1, 1], [3, 20], [70, 1]])
def test_not_finite_q_stays_in_its_row(qa, f16, news):
    rng = np.random.default_rng(12)
    tables, pages = ref.tables_of(rng, [200 + news[0], 9 + news[1]], 16)
    pool = ref.pool_of(rng, 1, pages, 8, 16, f16)
    b = ref.Batch(qa, tables, [200, 9], news)
    q = rng.standard_normal((b.rows, 16, 128)).astype(np.float32)
    q[0, 3, 7], q[0, 4, 0], q[-1, 9, 100] = np.nan, np.inf, -np.inf
    got = ref.run_attention(qa, q.reshape(b.rows, -1), pool, 0, b, 16, 16)
    want = ref.attention(q, pool, 0, tables, 16, b.past, b.start, 16)
    bad = np.isnan(want)
    assert bad[0, 3].all() and bad.sum() >= 2 * 128
    assert np.array_equal(np.isnan(got), bad)
    close(got[~bad], want[~bad], np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("max_len", [1, 300, 100000])
@pytest.mark.parametrize("news", [[1, 1], [90, 1]])
def test_max_len_is_a_hint(qa, f16, max_len, news):
    """The last key range takes whatever lies behind the host's bound."""
    rng = np.random.default_rng(max_len)
    past = [900, 20]
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], 32)
    pool = ref.pool_of(rng, 1, pages, 8, 32, f16)
    b = ref.Batch(qa, tables, past, news, max_len=max_len)
    q = rng.standard_normal((b.rows, 2048)).astype(np.float32)
    got = ref.run_attention(qa, q, pool, 0, b, 32, 16)
    close(got, ref.attention(q, pool, 0, tables, 32, b.past, b.start, 16), np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past", [-3, -(2 ** 31), 2 ** 31 - 1, 2 ** 30])
@pytest.mark.parametrize("new", [2, 50])
def test_positions_outside_every_table(qa, f16, past, new):
    """Tokens before position 0 see nothing; tokens behind the table row see all of it."""
    rng = np.random.default_rng(1)
    tables, pages = ref.tables_of(rng, [48, 20], 16, extra=0)
    pool = ref.pool_of(rng, 1, pages, 8, 16, f16)
    b = ref.Batch(qa, tables, [past, 19], [new, 1], max_len=64)
    q = rng.standard_normal((b.rows, 2048)).astype(np.float32)
    got = ref.run_attention(qa, q, pool, 0, b, 16, 16, fill=2.0)
    want = ref.attention(q, pool, 0, tables, 16, [int(past), 19], b.start, 16)
    if past > 0:
        assert (want[:new] != 0).all()
    close(got, want, np.abs(pool.astype(np.float64)).max())


def test_cache_beyond_32_bit_offsets(qa):
    """Pages whose K rows lie 3 GB and whose V rows lie 6 GB into the cache: append, attention and copies reach them."""
    page, pages = 16, 100000
    lay = ref.layout(qa, 1, pages, 8, page, True)
    total = qa.lib.qa_kv_cache_bytes(C.byref(lay))
    assert total > 6 << 30
    block = 8 * page * 128 * 2
    base = C.c_void_p()
    qa.check(qa.lib.qa_device_malloc(C.byref(base), total))
    try:
        def at(kv, p):
            return C.c_void_p(base.value + (kv * pages + int(p)) * block)

        rng = np.random.default_rng(2)
        past, new = [50, 30], [1, 40]
        small, count = ref.tables_of(rng, [51, 70], page, spare=0)
        place = pages - 1 - rng.permutation(400)[:count]              # the last pages of the cache
        place[0] = pages - 1
        tables = np.where(small >= 0, place[np.maximum(small, 0)], -1).astype(np.int32)
        pool = ref.pool_of(rng, 1, count, 8, page, True)
        for i, p in enumerate(place):
            for kv in (0, 1):
                rows = np.ascontiguousarray(pool[0, kv, i])
                qa.check(qa.lib.qa_copy_to_device(at(kv, p), rows.ctypes.data, block))
        b = ref.Batch(qa, tables, past, new)
        qkv = rng.standard_normal((41, 4096)).astype(np.float32)
        w = np.ones(128, np.float32)
        d = [qa.DeviceArray.from_numpy(a) for a in (qkv, w, w)]
        q, out = qa.DeviceArray((41, 2048)), qa.DeviceArray((41, 2048))
        qa.check(qa.lib.qa_paged_append(*(x.ptr for x in d), q.ptr, base, C.byref(lay), 0, b.ref, 16, 1e6, 1e-6, None))
        qa.check(qa.lib.qa_paged_attn(q.ptr, base, C.byref(lay), 0, b.ref, 16, ref.SCALE, out.ptr, None, 0, None))
        src, dst = int(tables[1, 3]), 7                               # and back into the first pages
        pair = [qa.DeviceArray.from_numpy(np.array([v], np.int32)) for v in (src, dst)]
        qa.check(qa.lib.qa_pages_copy(base, C.byref(lay), pair[0].ptr, pair[1].ptr, 1, None))
        qa.synchronize()
        for i, p in enumerate(place):
            for kv in (0, 1):
                qa.check(qa.lib.qa_copy_to_host(pool[0, kv, i].ctypes.data, at(kv, p), block))
        np.testing.assert_array_equal(pool[0, 1, small[1, 4], :, 5], qkv[40, 3 * 1024:].reshape(8, 128).astype(np.float16))
        copied = np.empty((8, page, 128), np.float16)
        qa.check(qa.lib.qa_copy_to_host(copied.ctypes.data, at(1, dst), block))
        np.testing.assert_array_equal(copied, pool[0, 1, small[1, 3]])
        want = ref.attention(q.numpy(), pool, 0, small, page, b.past, b.start, 16)
        close(out.numpy().reshape(want.shape), want, np.abs(pool.astype(np.float64)).max())
    finally:
        qa.lib.qa_device_free(base)


# ------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past,news,page", [([0], [1], 16), ([15, 16, 200], [1, 1, 1], 16), ([3, 0, 60], [40, 0, 5], 32),
                                            ([4000], [3], 256), ([10], [300], 64)])
def test_append(qa, f16, past, news, page):
    rng = np.random.default_rng(len(past) + past[0])
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], page)
    pool = ref.pool_of(rng, 3, pages, 8, page, f16)
    b = ref.Batch(qa, tables, past, news, n_rows=sum(news) + 2)
    qkv = rng.standard_normal((b.rows, 4096)).astype(np.float32)
    qn, kn = ((1 + 0.1 * rng.standard_normal(128)).astype(np.float32) for _ in range(2))
    lay = ref.layout(qa, 3, pages, 8, page, f16)
    d = [qa.DeviceArray.from_numpy(a) for a in (qkv, qn, kn, np.full((b.rows, 2048), 3.5, np.float32), pool)]
    print(f"append past={past} news={news} page={page} f16={f16}", flush=True)
    qa.check(qa.lib.qa_paged_append(*(x.ptr for x in d), C.byref(lay), 1, b.ref, 16, 1e6, 1e-6, None))
    qa.synchronize()
    q, got = d[3].numpy(), d[4].numpy()
    assert (q[sum(news):] == 3.5).all()
    step = 2.0 ** -11 if f16 else 0.0
    expect = pool.astype(np.float64)
    for s in range(len(past)):
        for r in range(b.start[s], b.start[s + 1]):
            pos = past[s] + r - b.start[s]
            x = qkv[r].reshape(32, 128)
            wq, wk = ref.rope_norm(x[:16], qn, pos), ref.rope_norm(x[16:24], kn, pos)
            assert np.abs(q[r].reshape(16, 128) - wq).max() <= 2.0 ** -20 * np.abs(wq).max()
            pg, sl = tables[s, pos // page], pos % page
            expect[1, 0, pg, :, sl], expect[1, 1, pg, :, sl] = wk, x[24:]
            np.testing.assert_array_equal(got[1, 1, pg, :, sl], x[24:].astype(pool.dtype))
    assert (np.abs(got.astype(np.float64) - expect) <= np.abs(expect) * (step + 2.0 ** -22) + 2.0 ** -20 * 5).all()
    untouched = np.ones(got.shape, bool)
    for s in range(len(past)):
        for pos in range(past[s], past[s] + news[s]):
            untouched[1, :, tables[s, pos // page], :, pos % page] = False
    np.testing.assert_array_equal(got[untouched], pool[untouched])


@pytest.mark.parametrize("f16", [True, False])
def test_append_gives_the_bits_of_the_contiguous_append(qa, f16):
    rng = np.random.default_rng(1)
    T, past, page = 70, 45, 16
    qkv = rng.standard_normal((T, 4096)).astype(np.float32)
    qn, kn = ((1 + 0.1 * rng.standard_normal(128)).astype(np.float32) for _ in range(2))
    d = [qa.DeviceArray.from_numpy(a) for a in (qkv, qn, kn)]
    flat_lay = ref.layout(qa, 1, 1, 8, 128, f16)
    dt = np.float16 if f16 else np.float32
    flat, q0 = qa.DeviceArray((2, 8, 128, 128), dt), qa.DeviceArray((T, 2048))
    d_past = qa.DeviceArray.from_numpy(np.array([past], np.int32))
    qa.check(qa.lib.qa_kv_append(*(x.ptr for x in d), q0.ptr, flat.ptr, C.byref(flat_lay), 0, d_past.ptr, 1, T, 16, 1e6, 1e-6, None))
    tables, pages = ref.tables_of(rng, [past + T], page)
    b = ref.Batch(qa, tables, [past], [T])
    lay = ref.layout(qa, 1, pages, 8, page, f16)
    pool, q1 = qa.DeviceArray((2, pages, 8, page, 128), dt), qa.DeviceArray((T, 2048))
    qa.check(qa.lib.qa_paged_append(*(x.ptr for x in d), q1.ptr, pool.ptr, C.byref(lay), 0, b.ref, 16, 1e6, 1e-6, None))
    qa.synchronize()
    np.testing.assert_array_equal(q0.numpy().view(np.uint32), q1.numpy().view(np.uint32))
    a, p = flat.numpy(), pool.numpy()
    for pos in range(past, past + T):
        np.testing.assert_array_equal(a[:, :, pos], p[:, tables[0, pos // page], :, pos % page])


def test_append_drops_positions_without_a_page(qa):
    rng = np.random.default_rng(4)
    tables = np.array([[1, -1, 9], [2 ** 31 - 1, 0, -7]], np.int32)     # 4 pages
    pool = ref.pool_of(rng, 1, 4, 8, 16, True)
    news = [60, 20]                                                     # the first sequence outgrows its row, too
    b = ref.Batch(qa, tables, [0, 0], news)
    qkv = rng.standard_normal((80, 4096)).astype(np.float32)
    w = np.ones(128, np.float32)
    lay = ref.layout(qa, 1, 4, 8, 16, True)
    d = [qa.DeviceArray.from_numpy(a) for a in (qkv, w, w, np.zeros((80, 2048), np.float32), pool)]
    qa.check(qa.lib.qa_paged_append(*(x.ptr for x in d), C.byref(lay), 0, b.ref, 16, 1e6, 1e-6, None))
    qa.synchronize()
    got = d[4].numpy()
    np.testing.assert_array_equal(got[:, :, 2:], pool[:, :, 2:])
    np.testing.assert_array_equal(got[0, 1, 1].transpose(1, 0, 2), qkv[:16, 3 * 1024:].reshape(16, 8, 128).astype(np.float16))
    np.testing.assert_array_equal(got[0, 1, 0, :, :4].transpose(1, 0, 2), qkv[76:80, 3 * 1024:].reshape(4, 8, 128).astype(np.float16))
    np.testing.assert_array_equal(got[0, 1, 0, :, 4:], pool[0, 1, 0, :, 4:])
    assert (d[3].numpy() != 0).any(axis=1).all()                        # q of every row all the same
