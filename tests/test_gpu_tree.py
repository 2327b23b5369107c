"""Drafted trees over a paged cache: masks, append, attention, acceptance and the accepted rows, against plain 64-bit statements.

Tolerances: those of causal attention over the same caches (products and sums are f32: 5e-6 in the 2-norm, 2^-16 of the largest
|v| for one value); q of an append within 2^-20 of its row's largest value; everything else is whole numbers or moved bytes."""
import ctypes as C

import numpy as np
import pytest

import candidates_ref as cand
import paged_ref as ref
from test_gpu_q8_cache import appended, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


def case(qa, seed, cache, past, news, page, kv_heads=8, group=2, mask=None, words=None, n_rows=None, fill=0.0, holes=(), change=None,
         roots=0.0, workspace=None, reach=5, **bounds):
    rng = np.random.default_rng(seed)
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], page)
    for s, j, to in holes:
        tables[s, j] = to
    pool = cand.Pool(qa, cache, 2, pages, kv_heads, page, rng)
    if change:
        change(pool, tables)
    heads = kv_heads * group
    b = ref.Batch(qa, tables, past, news, n_rows=n_rows, **bounds)
    if mask is None:
        parents = np.concatenate([cand.random_tree(rng, n, reach, roots) for n in news] + [np.full(b.rows - sum(news), -1, np.int32)])
        mask, _ = cand.masks_of(parents, b.start, b.rows, words or -(-max(news + [1]) // 32))
    q = rng.standard_normal((b.rows, heads * 128)).astype(np.float32)
    print(f"tree attention {cache} past={past} news={news} page={page} kv_heads={kv_heads} group={group} words={mask.shape[1]}", flush=True)
    got = cand.run_attention(qa, q, pool, 1, b, heads, mask=mask, fill=fill, workspace=workspace)
    want = cand.tree_attention(q, pool.values, 1, tables, page, b.past, b.start, heads, mask, out=np.full((b.rows, heads, 128), fill))
    return got, want, pool, b


@pytest.mark.parametrize("cache", cand.CACHES)
@pytest.mark.parametrize("past,news,page", [
    ([0], [1], 16), ([0], [8], 16), ([156], [8], 16), ([15], [4], 16), ([16], [17], 32), ([31, 0, 700], [33, 5, 1], 16),
    ([100, 3, 60, 0], [1, 64, 0, 65], 64), ([1000], [130], 128), ([3900], [9], 16), ([700, 1037], [63, 58], 16), ([2700], [290], 32),
    ([5], [300], 16),
])
def test_attention(qa, cache, past, news, page):
    got, want, pool, _ = case(qa, 3 + past[0], cache, past, news, page)
    close(got, want, np.abs(pool.values).max())


@pytest.mark.parametrize("cache", cand.CACHES)
@pytest.mark.parametrize("kv_heads,group,news", [(1, 1, 20), (2, 3, 1), (2, 3, 37), (4, 8, 1), (3, 16, 2), (8, 1, 8), (5, 5, 3), (8, 4, 2)])
def test_head_layouts(qa, cache, kv_heads, group, news):
    got, want, pool, _ = case(qa, 8, cache, [50, 9], [news, 1], 32, kv_heads=kv_heads, group=group)
    close(got, want, np.abs(pool.values).max())


@pytest.mark.parametrize("cache", cand.CACHES)
@pytest.mark.parametrize("past,news", [([40], [40]), ([0, 0], [20, 33]), ([2700], [280])])
def test_any_mask(qa, cache, past, news):
    """Masks of no tree: random bits, rows that see no new token, not even themselves, bits behind the sequence's rows."""
    rng = np.random.default_rng(4)
    words = -(-max(news) // 32) + 1
    mask = rng.integers(0, 2 ** 32, (sum(news), words), dtype=np.uint64).astype(np.uint32)
    mask[::7] = 0
    mask[1::7] = 0xffffffff
    got, want, pool, _ = case(qa, 5, cache, past, news, 16, mask=mask)
    close(got, want, np.abs(pool.values).max())
    if past[0] == 0:
        assert (got[0] == 0).all()


@pytest.mark.parametrize("cache", cand.CACHES)
def test_a_full_lower_triangle_is_causal_attention(qa, cache):
    n = 70
    mask = np.zeros((n, 3), np.uint32)
    for i in range(n):
        for j in range(i + 1):
            mask[i, j // 32] |= np.uint32(1 << (j % 32))
    got, want, pool, b = case(qa, 6, cache, [90], [n], 16, mask=mask)
    close(got, want, np.abs(pool.values).max())


@pytest.mark.parametrize("cache", cand.CACHES)
def test_masks_shorter_than_the_sequences(qa, cache):
    """Nodes behind 32 mask_words are seen by nobody."""
    got, want, pool, _ = case(qa, 7, cache, [20, 0], [50, 90], 16, words=1)
    close(got, want, np.abs(pool.values).max())


@pytest.mark.parametrize("cache", cand.CACHES)
@pytest.mark.parametrize("past,news,holes", [([60], [10], [(0, 1, -1)]), ([20], [20], [(0, 0, -1), (0, 1, -1), (0, 2, -1)]),
                                             ([16], [20], [(0, 0, -1), (0, 1, -7)]), ([2700], [290], [(0, j, -1) for j in range(2, 180, 9)])])
def test_positions_without_a_page(qa, cache, past, news, holes):
    got, want, pool, _ = case(qa, 9, cache, past, news, 16, holes=holes, fill=3.0)
    close(got, want, np.abs(pool.values).max())


@pytest.mark.parametrize("cache", cand.CACHES)
@pytest.mark.parametrize("past,news", [([37], [12]), ([0], [40]), ([2700], [280])])
def test_what_siblings_hold_does_not_matter(qa, cache, past, news):
    """K and V of a node that only its children see are NaN: every other row is as it should be."""
    rng = np.random.default_rng(0)
    n = news[0]
    parents = cand.random_tree(rng, n)
    bad = n // 2
    lines = cand.ancestors(parents)
    sees = np.array([bad in line for line in lines])
    start = np.array([0, n])
    mask, _ = cand.masks_of(parents, start, n, -(-n // 32))

    def change(pool, tables):
        pg, sl = tables[0, (past[0] + bad) // 16], (past[0] + bad) % 16
        if cache == "q8":
            pool.scales[:, :, pg, :, sl] = np.nan
        else:
            pool.raw[:, 0, pg, :, sl] = np.inf
            pool.raw[:, 1, pg, :, sl] = np.nan
    got, want, pool, _ = case(qa, 11, cache, past, news, 16, mask=mask, change=change)
    assert np.isnan(got[sees]).all() and sees.any() and not sees.all()
    close(got[~sees], want[~sees], 6.0)


FILLING = [([1600, 900, 1300, 40, 700], [41, 36, 31, 26, 21]), ([2000, 1700], [32, 27]), ([700] * 11 + [300], [24, 3] * 5 + [0, 30]),
           ([500, 30, 900, 100, 250, 31, 0, 64, 200], [40, 4, 3, 1, 4, 2, 4, 1, 3])]


@pytest.mark.parametrize("cache", cand.CACHES)
@pytest.mark.parametrize("past,news", FILLING)
@pytest.mark.parametrize("page,holes", [(16, ()), (64, [(0, 0, -1), (1, 2, 1 << 30), (0, 7, -1)])])
def test_trees_that_fill_the_chip(qa, cache, past, news, page, holes):
    got, want, pool, _ = case(qa, 14, cache, past, news, page, holes=[h for h in holes if h[1] * page < past[h[0]] + news[h[0]]])
    close(got, want, np.abs(pool.values).max())


@pytest.mark.parametrize("cache", cand.CACHES)
@pytest.mark.parametrize("past,news", FILLING)
def test_any_mask_where_trees_fill_the_chip(qa, cache, past, news):
    """Random masks, the cached positions not finite in a page that no table holds."""
    rng = np.random.default_rng(15)
    mask = rng.integers(0, 2 ** 32, (sum(news), 2), dtype=np.uint64).astype(np.uint32)
    mask[::5] = 0

    def change(pool, tables):
        free = np.setdiff1d(np.arange(pool.raw.shape[2] if cache != "q8" else pool.scales.shape[2]), tables)
        if cache == "q8":
            pool.scales[:, :, free] = np.nan
        else:
            pool.raw[:, :, free] = np.nan
    got, want, pool, _ = case(qa, 16, cache, past, news, 16, mask=mask, change=change)
    close(got, want, 6.0)


def test_rows_of_no_sequence_and_no_bounds(qa):
    got, want, pool, b = case(qa, 12, "f16", [40, 0, 300], [9, 20, 1], 16, n_rows=33, fill=2.5, max_tokens=0, max_len=0)
    close(got[:30], want[:30], np.abs(pool.values).max())
    assert (got[30:] == 2.5).all()


def test_less_workspace(qa):
    for cache in cand.CACHES:
        got, want, pool, _ = case(qa, 13, cache, [3800], [20], 16, workspace=0)
        close(got, want, np.abs(pool.values).max())


# ------------------------------------------------------------------------------------------ bookkeeping
def prepared(qa, parents, start, rows, words):
    tables = np.full((len(start) - 1, 1), -1, np.int32)
    b = ref.Batch(qa, tables, [0] * (len(start) - 1), np.diff(start).tolist(), n_rows=rows)
    b.d[2].upload(np.asarray(start, np.int32))
    mask, depth = qa.DeviceArray.from_numpy(np.full((rows, words), 77, np.int32)), qa.DeviceArray.from_numpy(np.full(rows, 77, np.int32))
    d_par = qa.DeviceArray.from_numpy(np.asarray(parents, np.int32))
    qa.check(qa.lib.qa_tree_prepare(b.ref, d_par.ptr, mask.ptr, words, depth.ptr, None))
    qa.synchronize()
    return mask.numpy().view(np.uint32), depth.numpy()


@pytest.mark.parametrize("news,words,reach,roots", [([1], 1, 1, 0), ([8], 1, 5, 0), ([33, 0, 64, 65], 3, 4, 0.1), ([1000], 32, 3, 0.01), ([1024], 32, 1, 0),
                                                    ([200], 2, 7, 0), ([5] * 150, 1, 2, 0.3)])
def test_prepare(qa, news, words, reach, roots):
    rng = np.random.default_rng(len(news) + words)
    start = np.concatenate([[0], np.cumsum(news)])
    parents = np.concatenate([cand.random_tree(rng, n, reach, roots) for n in news]).astype(np.int32)
    mask, depth = prepared(qa, parents, start, len(parents), words)
    want, want_depth = cand.masks_of(parents, start, len(parents), words)
    np.testing.assert_array_equal(mask, want)
    np.testing.assert_array_equal(depth, want_depth)


def test_prepare_of_parents_that_are_none(qa):
    """A parent that is not a lower number is none; rows before and behind the sequences, and nodes behind 1024, are left alone."""
    start = np.array([2, 7])
    parents = np.array([0, 0, 5, -1, 1, 2 ** 31 - 1, 3, 0, 0], np.int32)
    mask, depth = prepared(qa, parents, start, 9, 2)
    assert (mask[[0, 1, 7, 8]] == 77).all() and (depth[[0, 1, 7, 8]] == 77).all()
    assert mask[2:7].tolist() == [[1, 0], [2, 0], [6, 0], [8, 0], [24, 0]] and depth[2:7].tolist() == [0, 0, 1, 0, 1]
    parents = np.arange(-1, 1029, dtype=np.int32)
    mask, depth = prepared(qa, parents, np.array([0, 1030]), 1030, 32)
    assert depth[:1024].tolist() == list(range(1024)) and (depth[1024:] == 77).all() and (mask[1024:] == 77).all()
    assert (mask[1023] == 0xffffffff).all()


def accepted(qa, parents, ids, picks, start, rows):
    n = len(start) - 1
    b = ref.Batch(qa, np.full((n, 1), -1, np.int32), [0] * n, np.diff(start).tolist(), n_rows=rows)
    b.d[2].upload(np.asarray(start, np.int32))
    d = [qa.DeviceArray.from_numpy(np.asarray(a, np.int32)) for a in (parents, ids, picks)]
    path = qa.DeviceArray.from_numpy(np.full(rows, 55, np.int32))
    kept, nxt = qa.DeviceArray((n,), np.int32), qa.DeviceArray((n,), np.int32)
    qa.check(qa.lib.qa_tree_accept(b.ref, d[0].ptr, d[1].ptr, d[2].ptr, path.ptr, kept.ptr, nxt.ptr, None))
    qa.synchronize()
    return path.numpy(), kept.numpy(), nxt.numpy()


@pytest.mark.parametrize("news", [[1], [8], [41, 0, 3, 64], [1024], [7] * 150, [1000, 1]])
@pytest.mark.parametrize("ids_of", [2, 50])
def test_accept(qa, news, ids_of):
    """Few ids: several children hold the picked one, and the first is taken."""
    rng = np.random.default_rng(len(news) + ids_of)
    start = np.concatenate([[0], np.cumsum(news)])
    parents = np.concatenate([cand.random_tree(rng, n, 3) for n in news]).astype(np.int32)
    rows = len(parents)
    ids, picks = rng.integers(0, ids_of, rows).astype(np.int32), rng.integers(0, ids_of, rows).astype(np.int32)
    path, kept, nxt = accepted(qa, parents, ids, picks, start, rows)
    for s, n in enumerate(news):
        lo, hi = start[s], start[s + 1]
        if n == 0:
            assert kept[s] == 0 and nxt[s] == -1
            continue
        want, last = cand.accept(parents[lo:hi], ids[lo:hi], picks[lo:hi])
        assert kept[s] == len(want) and nxt[s] == last
        assert path[lo:hi].tolist() == want + [-1] * (n - len(want))


def keep(qa, pool, tables, past, news, path, kept, rows=None):
    b = ref.Batch(qa, tables, past, news, n_rows=rows)
    d_pool = pool.upload()
    d = [qa.DeviceArray.from_numpy(np.asarray(a, np.int32)) for a in (path, kept)]
    qa.check(qa.lib.qa_paged_keep(d_pool.ptr, C.byref(pool.layout), b.ref, d[0].ptr, d[1].ptr, None))
    qa.synchronize()
    return pool.take(d_pool.numpy())


def moved(pool, tables, page, past, starts, path, n_moved):
    """The pool's arrays after the moves, one row after another in order."""
    arrays = [a.copy() for a in ((pool.ints, pool.scales) if pool.cache == "q8" else (pool.raw,))]
    for s, n in enumerate(n_moved):
        for k in range(n):
            a, b = past[s] + path[starts[s] + k], past[s] + k
            ends = [tables[s, x // page] if x // page < tables.shape[1] else -1 for x in (a, b)]
            if any(not 0 <= e < pool.layout.n_streams for e in ends):
                continue
            for x in arrays:
                x[:, :, ends[1], :, b % page] = x[:, :, ends[0], :, a % page]
    return arrays


@pytest.mark.parametrize("cache", cand.CACHES)
@pytest.mark.parametrize("past,news,page,kv_heads", [([0], [1], 16, 8), ([156], [8], 16, 8), ([10, 0, 31], [41, 20, 64], 16, 8), ([200, 7], [150, 3], 32, 3),
                                                     ([5], [60], 64, 20), ([3], [1024], 16, 1), ([40], [300], 256, 8)])
def test_keep(qa, cache, past, news, page, kv_heads):
    rng = np.random.default_rng(sum(news))
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], page)
    pool = cand.Pool(qa, cache, 2, pages, kv_heads, page, rng)
    starts = np.concatenate([[0], np.cumsum(news)])
    path, kept = np.full(starts[-1], -1, np.int32), []
    for s, n in enumerate(news):
        chosen = np.flatnonzero(rng.random(n) < 0.6)
        path[starts[s]:starts[s] + len(chosen)] = chosen
        kept.append(len(chosen))
    got = keep(qa, pool, tables, past, news, path, kept)
    want = moved(pool, tables, page, past, starts, path, kept)
    for a, b in zip((got.ints, got.scales) if cache == "q8" else (got.raw,), want):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_keep_of_what_is_no_path(qa, cache):
    """Entries that do not rise or are no node end a path; places without a page are passed over; too many kept are no more than the rows."""
    rng = np.random.default_rng(1)
    news, past = [9, 9, 9, 9, 9], [20, 30, 12, 8, 4]
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], 16)
    tables[3, 0] = -1
    tables[3, 1] = pages
    pool = cand.Pool(qa, cache, 1, pages, 2, 16, rng)
    paths = [[0, 3, 3, 5], [2, 1, 5, 6], [1, 2, 9, 10], [3, 5, 6, 8], [1, 2, 4, 5, 6, 7, 8]]
    path = np.full(45, -1, np.int32)
    for s, p in enumerate(paths):
        path[9 * s:9 * s + len(p)] = p
    got = keep(qa, pool, tables, past, news, path, [4, 4, 4, 4, 2 ** 31 - 1])
    want = moved(pool, tables, 16, past, np.arange(0, 50, 9), path, [2, 1, 2, 4, 7])
    for a, b in zip((got.ints, got.scales) if cache == "q8" else (got.raw,), want):
        np.testing.assert_array_equal(a, b)
    got = keep(qa, pool, tables, past, news, path, [0, -5, 0, 0, 0])
    np.testing.assert_array_equal(got.bytes(), pool.bytes())


@pytest.mark.parametrize("cache", cand.CACHES)
def test_append_with_depths(qa, cache):
    """Rows lie at n_past + their number and are turned by n_past + their depth."""
    rng = np.random.default_rng(3)
    past, news = [100, 0], [12, 30]
    parents = np.concatenate([cand.random_tree(rng, n) for n in news])
    start = np.array([0, 12, 42])
    _, depth = cand.masks_of(parents, start, 42, 1)
    q, old, pool, out, b, tables, qkv, wq, wk = appended(qa, cache, past, news, 16, depth=depth)
    x = qkv.reshape(42, 32, 128)
    for r in range(42):
        s = 0 if r < 12 else 1
        want = ref.rope_norm(x[r, :16], wq, past[s] + depth[r])
        assert np.abs(q[r] - want).max() <= 2.0 ** -20 * np.abs(want).max()
        k = ref.rope_norm(x[r, 16:24], wk, past[s] + depth[r])
        pos = past[s] + r - start[s]
        got = pool.values[1, 0, tables[s, pos // 16], :, pos % 16]
        size = np.abs(k).max(-1, keepdims=True)
        half = {"f32": 0.0, "f16": 2.0 ** -11, "q8": 0.5 / 127}[cache]
        assert (np.abs(got - k) <= (half + 2.0 ** -20 + (cache == "q8") * 2.0 ** -12 / 127) * size).all()
    # as deep as they are far: the plain append, bit by bit
    flat = np.concatenate([np.arange(n) for n in news])
    a = appended(qa, cache, past, news, 16, depth=flat)
    c = appended(qa, cache, past, news, 16)
    np.testing.assert_array_equal(a[0], c[0])
    np.testing.assert_array_equal(a[2].bytes(), c[2].bytes())
