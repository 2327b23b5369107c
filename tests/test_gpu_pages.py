"""Bookkeeping of pages on the device against plain statements that walk the lists entry by entry: whole numbers and moved
rows are equal."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


class Pool:
    """Pages, counts and tables on the device."""

    def __init__(self, qa, refs, tables, page=16, layers=2, heads=2, f16=True, seed=0):
        self.qa, self.page, self.f16 = qa, page, f16
        self.refs, self.tables = np.asarray(refs, np.int32), np.asarray(tables, np.int32)
        self.host = ref.pool_of(np.random.default_rng(seed), layers, len(self.refs), heads, page, f16)
        self.lay = ref.layout(qa, layers, len(self.refs), heads, page, f16)
        self.d_pool, self.d_refs, self.d_tables = (qa.DeviceArray.from_numpy(a) for a in (self.host, self.refs, self.tables))
        self.ws_bytes = qa.lib.qa_pages_workspace_bytes(C.byref(self.lay))
        self.ws = qa.DeviceArray.from_numpy(np.full(self.ws_bytes, 0xff, np.uint8))
        self.keep = []

    def ints(self, values):
        if values is None:
            return None
        self.keep.append(self.qa.DeviceArray.from_numpy(np.asarray(values, np.int32)))
        return self.keep[-1].ptr

    def counts(self):
        return self.d_refs.ptr, len(self.refs), self.d_tables.ptr, self.tables.shape[0], self.tables.shape[1], self.page

    def extend(self, rows, past, new, stream=None):
        missing = self.qa.DeviceArray.from_numpy(np.array([-99], np.int32))
        self.qa.check(self.qa.lib.qa_pages_extend(self.d_pool.ptr, C.byref(self.lay), self.d_refs.ptr, self.d_tables.ptr,
                                                  self.tables.shape[0], self.tables.shape[1], self.ints(rows), self.ints(past),
                                                  self.ints(new), len(past), missing.ptr, self.ws.ptr, self.ws_bytes, stream))
        self.qa.synchronize()
        return int(missing.numpy()[0])

    def state(self):
        return self.d_refs.numpy(), self.d_tables.numpy(), self.d_pool.numpy()

    def same(self, refs, tables, pool):
        r, t, p = self.state()
        np.testing.assert_array_equal(r, refs)
        np.testing.assert_array_equal(t, tables)
        np.testing.assert_array_equal(p.view(np.uint8), pool.view(np.uint8))


def counted(tables, pages):
    t = np.asarray(tables)
    return np.bincount(t[(t >= 0) & (t < pages)], minlength=pages).astype(np.int32)


def check_extend(qa, pool, rows, past, new):
    refs, tables, copies, missing = ref.extend(pool.refs, pool.tables, pool.page, rows if rows is not None else range(len(past)), past, new)
    host = pool.host.copy()
    for a, b in copies:
        host[:, :, b] = pool.host[:, :, a]
    assert pool.extend(rows, past, new) == missing
    pool.same(refs, tables, host)
    return copies, missing


@pytest.mark.parametrize("f16,page", [(True, 16), (False, 16), (True, 64), (False, 256)])
def test_extend_copies_what_is_shared(qa, f16, page):
    """Three rows share a partly filled page and are written at once: two copies, the last holder keeps it."""
    tables = np.full((4, 5), -1, np.int32)
    tables[0:3, 0], tables[0:3, 1] = 4, 2
    tables[3, 0] = 0
    pool = Pool(qa, counted(tables, 12), tables, page=page, f16=f16)
    at = page + page // 2
    copies, missing = check_extend(qa, pool, None, [at, at, at, 1], [1, page, 2 * page, 1])
    assert copies == [(2, 1), (2, 3)] and missing == 0


def test_extend_one_of_two_holders(qa):
    tables = np.array([[3, 1, -1], [3, 1, -1]], np.int32)
    pool = Pool(qa, counted(tables, 6), tables)
    copies, _ = check_extend(qa, pool, [1], [20], [5])
    assert copies == [(1, 0)]


def test_extend_at_a_page_border_takes_new_pages_only(qa):
    tables = np.array([[3, 1, -1, -1], [3, 1, -1, -1]], np.int32)
    pool = Pool(qa, counted(tables, 9), tables)
    copies, _ = check_extend(qa, pool, None, [32, 32], [1, 17])
    assert copies == []


@pytest.mark.parametrize("rows,past,new", [
    ([5, -1, 0, 2 ** 31 - 1], [0, 0, 0, 0], [3, 3, 3, 3]),      # numbers outside the table
    ([1, 1, 0], [0, 40, 0], [3, 9, 50]),                        # a row twice: the second time left out
    ([0, 1], [-1, 5], [9, 0]), ([0, 1], [0, 2 ** 31 - 1], [-4, 3]),   # nothing to provide
    ([0], [60], [2 ** 31 - 1]), ([1], [500], [10]),             # behind the table row
    ([0, 1, 2], [0, 0, 0], [64, 64, 64]),                       # more than there are
])
def test_extend_odd_lists(qa, rows, past, new):
    tables = np.full((3, 4), -1, np.int32)
    tables[0, 0] = 5
    pool = Pool(qa, counted(tables, 9), tables)
    check_extend(qa, pool, rows, past, new)


def test_extend_all_or_nothing(qa):
    tables = np.array([[0, 1, -1, -1], [0, 1, -1, -1], [2, -1, -1, -1]], np.int32)
    pool = Pool(qa, counted(tables, 5), tables)
    _, missing = check_extend(qa, pool, None, [20, 20, 16], [20, 30, 1])
    assert missing == 3          # a copy and one page (positions to 39), two pages (to 49), one page: five, two are free
    enough = Pool(qa, np.r_[pool.refs, 0, 0, 0], tables)
    assert check_extend(qa, enough, None, [20, 20, 16], [20, 30, 1])[1] == 0


def test_extend_entries_outside_the_cache_count_as_none(qa):
    tables = np.array([[2, 77, -9, 3], [4, 2 ** 31 - 1, -1, -1]], np.int32)
    pool = Pool(qa, counted(tables, 9), tables)
    check_extend(qa, pool, None, [10, 10], [54, 40])


@pytest.mark.parametrize("n_pages", [1, 8191, 8192, 8193, 20000])
def test_extend_finds_the_lowest_free_pages(qa, n_pages):
    rng = np.random.default_rng(n_pages)
    refs = (rng.random(n_pages) < 0.97).astype(np.int32)
    refs[-1] = 0
    want = int((refs <= 0).sum())
    tables = np.full((4, max(1, want)), -1, np.int32)
    pool = Pool(qa, refs, tables, layers=1, heads=1)
    n = min(want, 60)
    check_extend(qa, pool, [2], [0], [16 * n])


def test_extend_many_rows(qa):
    """1024 list entries; most rows in pairs that share their last page."""
    rng = np.random.default_rng(5)
    n = 1024
    lens = rng.integers(1, 60, n // 2).repeat(2)
    counts = -(-lens // 16)
    tables, at = np.full((n, 8), -1, np.int32), 0
    for i in range(0, n, 2):
        tables[i, :counts[i]] = np.arange(at, at + counts[i])
        tables[i + 1] = tables[i]
        at += counts[i]
    pages = at + 3000
    order = rng.permutation(pages).astype(np.int32)
    tables = np.where(tables >= 0, order[np.maximum(tables, 0)], -1)
    pool = Pool(qa, counted(tables, pages), tables, layers=1, heads=1)
    rows = rng.permutation(n)
    check_extend(qa, pool, rows.tolist(), lens[rows].tolist(), rng.integers(0, 20, n).tolist())


def test_extend_of_nothing(qa):
    pool = Pool(qa, [1, 0], [[0]])
    assert pool.extend([], [], []) == 0
    pool.same(pool.refs, pool.tables, pool.host)


@pytest.mark.parametrize("src,dst,length", [
    ([0], [1], [40]), ([0, 0, 0], [1, 2, 3], [40, 16, 17]), ([0], [1], [0]), ([0], [1], [-5]), ([0], [1], [2 ** 31 - 1]),
    ([0], [0], [40]),                                    # onto itself
    ([0, 1], [1, 2], [40, 40]),                          # a dst that is read: left out
    ([0, 3, 0], [2, 2, 2], [40, 20, 33]),                # the same dst: the last one
    ([0, 9, -1], [7, 1, 2], [40, 40, 40]),               # outside the table
])
def test_fork(qa, src, dst, length):
    tables = np.array([[0, 5, 2, -1], [7, 8, -1, -1], [0, 99, -1, -1], [3, -1, -1, -1]], np.int32)
    pool = Pool(qa, counted(tables, 10), tables)
    refs, want = ref.fork(pool.refs, tables, 16, src, dst, length)
    qa.check(qa.lib.qa_pages_fork(*pool.counts(), pool.ints(src), pool.ints(dst), pool.ints(length), len(src), None))
    qa.synchronize()
    pool.same(refs, want, pool.host)


@pytest.mark.parametrize("rows,keep", [([1], None), ([0, 2], [16, 17]), ([2, 2, 1], [40, 3, 0]), ([9, -1, 0], [0, 0, 1]),
                                       ([0], [2 ** 31 - 1]), ([0], [-7])])
def test_free(qa, rows, keep):
    tables = np.array([[0, 5, 2, -1], [0, 5, 44, -3], [0, 6, 3, 1]], np.int32)
    pool = Pool(qa, counted(tables, 8), tables)
    refs, want = ref.free(pool.refs, tables, 16, rows, keep or [0] * len(rows))
    qa.check(qa.lib.qa_pages_free(*pool.counts(), pool.ints(rows), pool.ints(keep), len(rows), None))
    qa.synchronize()
    pool.same(refs, want, pool.host)


@pytest.mark.parametrize("f16,page,heads", [(True, 16, 1), (False, 16, 3), (True, 256, 8), (False, 64, 5)])
def test_copy(qa, f16, page, heads):
    pool = Pool(qa, np.ones(9, np.int32), [[-1]], page=page, heads=heads, f16=f16, layers=3)
    src, dst = [0, 3, 5, -1, 2, 9, 8, 6], [1, 4, 5, 2, 2 ** 31 - 1, 7, 7, 4]
    host = pool.host.copy()
    for i, (a, b) in enumerate(zip(src, dst)):      # 3 -> 4 gives way to 6 -> 4, 9 -> 7 to 8 -> 7
        if 0 <= a < 9 and 0 <= b < 9 and a != b and b not in dst[i + 1:] and b not in src:
            host[:, :, b] = pool.host[:, :, a]
    assert (host[:, :, 4] == pool.host[:, :, 6]).all() and (host[:, :, 7] == pool.host[:, :, 8]).all()
    qa.check(qa.lib.qa_pages_copy(pool.d_pool.ptr, C.byref(pool.lay), pool.ints(src), pool.ints(dst), len(src), None))
    qa.synchronize()
    pool.same(pool.refs, pool.tables, host)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n_pages,used", [(1, 0.0), (1, 1.0), (2, 0.5), (50, 0.0), (50, 1.0), (50, 0.5), (300, 0.3), (700, 0.9), (20000, 0.6)])
def test_compact(qa, in_place, n_pages, used):
    rng = np.random.default_rng(n_pages)
    refs = np.where(rng.random(n_pages) < used, rng.integers(1, 4, n_pages), rng.integers(-1, 1, n_pages)).astype(np.int32)
    tables = rng.integers(-2, n_pages + 2, (7, 19)).astype(np.int32)
    big = n_pages > 1000
    pool = Pool(qa, refs, tables, layers=1 if big else 3, heads=1 if big else 2)
    want_refs, want_tables, moves, live = ref.compact(refs, tables)
    host = pool.host.copy()
    for a, b in moves:
        host[:, :, b] = pool.host[:, :, a]
    d_live = qa.DeviceArray.from_numpy(np.array([-5], np.int32))
    r_out = pool.d_refs if in_place else qa.DeviceArray.from_numpy(np.full(n_pages, -77, np.int32))
    t_out = pool.d_tables if in_place else qa.DeviceArray.from_numpy(np.full(tables.shape, -77, np.int32))
    qa.check(qa.lib.qa_pages_compact(pool.d_pool.ptr, C.byref(pool.lay), pool.d_refs.ptr, pool.d_tables.ptr, 7, 19, r_out.ptr, t_out.ptr,
                                     d_live.ptr, pool.ws.ptr, pool.ws_bytes, None))
    qa.synchronize()
    assert int(d_live.numpy()[0]) == live
    np.testing.assert_array_equal(r_out.numpy(), want_refs)
    np.testing.assert_array_equal(t_out.numpy(), want_tables)
    np.testing.assert_array_equal(pool.d_pool.numpy().view(np.uint8), host.view(np.uint8))
    if not in_place:
        np.testing.assert_array_equal(pool.d_refs.numpy(), refs)
        np.testing.assert_array_equal(pool.d_tables.numpy(), tables)


def test_a_server_s_day(qa):
    """A seeded run of extend, fork, free and compact on one pool, each step compared; nobody's rows are lost or shared by
    mistake: every table's positions keep the values that its sequence has written."""
    rng = np.random.default_rng(11)
    n_rows, stride, page, n_pages = 6, 6, 16, 24
    pool = Pool(qa, np.zeros(n_pages, np.int32), np.full((n_rows, stride), -1, np.int32), page=page, layers=1, heads=1)
    refs, tables, host = pool.refs.copy(), pool.tables.copy(), pool.host.copy()
    length, content = [0] * n_rows, [[] for _ in range(n_rows)]
    stamp = 0
    for turn in range(60):
        kind = rng.choice(["extend", "extend", "extend", "fork", "free", "compact"])
        if kind == "extend":
            rows = rng.permutation(n_rows)[:3].tolist()
            new = [min(int(rng.integers(1, 20)), stride * page - length[r]) for r in rows]
            old = host.copy()
            refs, tables, copies, missing = ref.extend(refs, tables, page, rows, [length[r] for r in rows], new)
            for a, b in copies:
                host[:, :, b] = old[:, :, a]
            assert pool.extend(rows, [length[r] for r in rows], new) == missing
            if missing == 0:
                for r, n in zip(rows, new):
                    for _ in range(max(0, n)):
                        stamp += 1
                        host[:, :, tables[r, length[r] // page], :, length[r] % page] = stamp % 2000
                        content[r].append(stamp % 2000)
                        length[r] += 1
                pool.d_pool.upload(host)
        elif kind == "fork":
            a, b = rng.permutation(n_rows)[:2].tolist()
            n = int(rng.integers(0, length[a] + 1))
            refs, tables = ref.fork(refs, tables, page, [a], [b], [n])
            qa.check(qa.lib.qa_pages_fork(*pool.counts(), pool.ints([a]), pool.ints([b]), pool.ints([n]), 1, None))
            content[b], length[b] = content[a][:n], n
        elif kind == "free":
            r = int(rng.integers(0, n_rows))
            n = int(rng.integers(0, length[r] + 1)) if rng.random() < 0.5 else 0
            refs, tables = ref.free(refs, tables, page, [r], [n])
            qa.check(qa.lib.qa_pages_free(*pool.counts(), pool.ints([r]), pool.ints([n]), 1, None))
            content[r], length[r] = content[r][:n], n
        else:
            old = host.copy()
            refs, tables, moves, live = ref.compact(refs, tables)
            for a, b in moves:
                host[:, :, b] = old[:, :, a]
            d_live = qa.DeviceArray((1,), np.int32)
            qa.check(qa.lib.qa_pages_compact(pool.d_pool.ptr, C.byref(pool.lay), pool.d_refs.ptr, pool.d_tables.ptr, n_rows, stride,
                                             pool.d_refs.ptr, pool.d_tables.ptr, d_live.ptr, pool.ws.ptr, pool.ws_bytes, None))
            qa.synchronize()
            assert int(d_live.numpy()[0]) == live
        qa.synchronize()
        pool.same(refs, tables, host)
        np.testing.assert_array_equal(refs, counted(tables, n_pages))
        for r in range(n_rows):
            got = [host[0, 1, tables[r, j // page], 0, j % page, 0] for j in range(length[r])]
            assert got == content[r], (turn, kind, r)
