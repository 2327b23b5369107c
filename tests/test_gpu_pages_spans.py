"""qa_pages_extend where the positions that are about to be written reach over several pages that others hold: a sequence that
was forked, has gone back and goes on.  Every such page is made private, entry by entry in list order; counts, tables and
the bytes of every page are equal to a plain statement's, which walks the entries one by one."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as ref
from test_gpu_pages import Pool, counted
from test_gpu_paged_serving import Hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


def extend(refs, tables, page, rows, past, new):
    """(refs, tables, copies, missing): a copy for each written entry whose page has another holder left."""
    r, t = refs.copy(), tables.copy()
    free = [p for p in range(len(refs)) if refs[p] <= 0]
    copies, seen, need = [], set(), 0
    for row, n_past, n_new in zip(rows, past, new):
        if not 0 <= row < len(t) or n_new <= 0 or n_past < 0 or row in seen:
            continue
        seen.add(row)
        for j in range(n_past // page, min(t.shape[1], -(-(n_past + n_new) // page))):
            old = int(t[row, j])
            there = 0 <= old < len(r)
            if there and r[old] <= 1:
                continue
            if there:
                r[old] -= 1
            need += 1
            if need <= len(free):
                if there:
                    copies.append((old, free[need - 1]))
                t[row, j], r[free[need - 1]] = free[need - 1], 1
    return (r, t, copies, 0) if need <= len(free) else (refs.copy(), tables.copy(), [], need - len(free))


def check(qa, pool, rows, past, new):
    refs, tables, copies, missing = extend(pool.refs, pool.tables, pool.page, rows, past, new)
    host = pool.host.copy()
    for a, b in copies:
        host[:, :, b] = pool.host[:, :, a]
    print(f"extend {len(rows)} rows of {tables.shape}, {len(refs)} pages: {len(copies)} copies, {missing} missing", flush=True)
    assert pool.extend(rows, past, new) == missing
    pool.same(refs, tables, host)
    if missing == 0:
        for row, n_past, n_new in zip(rows, past, new):     # what is written is held once
            written = range(n_past // pool.page, min(tables.shape[1], -(-(n_past + n_new) // pool.page))) if n_new > 0 else ()
            assert all(refs[tables[row, j]] == 1 for j in written)
    return copies, missing


@pytest.mark.parametrize("f16,page", [(True, 16), (False, 16), (True, 256)])
@pytest.mark.parametrize("pages_back,new_pages", [(2, 2), (3, 5), (9, 3), (9, 12)])
def test_a_sequence_that_goes_back_over_shared_pages(qa, f16, page, pages_back, new_pages):
    """Row 1 shares ten pages with row 0, goes back and writes over them: row 0's pages keep their bytes."""
    tables = np.full((3, 24), -1, np.int32)
    tables[0, :10] = np.arange(10)[::-1] + 3
    tables[1] = tables[0]
    pool = Pool(qa, counted(tables, 40), tables, page=page, f16=f16)
    past = page * (10 - pages_back) + page // 2
    copies, _ = check(qa, pool, [1], [past], [new_pages * page])
    assert len(copies) == min(pages_back, new_pages + 1)
    before = pool.host[:, :, tables[0, :10]]
    np.testing.assert_array_equal(pool.d_pool.numpy()[:, :, pool.d_tables.numpy()[0, :10]], before)


@pytest.mark.parametrize("rows,past,new", [
    ([0, 1, 2], [20, 20, 20], [60, 60, 60]),          # all holders: the last one listed keeps its pages
    ([2, 0, 1], [20, 50, 33], [60, 1, 30]),           # from different positions on
    ([1, 0], [0, 79], [80, 1]), ([0, 1, 2], [0, 0, 0], [16, 16, 80]),
    ([1, 1, 0], [16, 0, 16], [33, 99, 33]),           # a row twice: the second time left out
    ([0, 7, 1], [16, 16, 16], [64, 64, 0]),
])
def test_holders_that_write_the_same_pages(qa, rows, past, new):
    tables = np.full((4, 7), -1, np.int32)
    tables[0:3, :5] = [4, 9, 2, 7, 0]
    tables[2, 4] = 11
    tables[3, 1] = 9
    pool = Pool(qa, counted(tables, 40), tables)
    refs, want, copies, missing = extend(pool.refs, tables, 16, rows, past, new)
    host = pool.host.copy()
    for a, b in copies:
        host[:, :, b] = pool.host[:, :, a]
    assert pool.extend(rows, past, new) == missing == 0
    pool.same(refs, want, host)


def test_all_or_nothing_counts_every_copy(qa):
    tables = np.array([[0, 1, 2, 3, -1], [0, 1, 2, 3, -1]], np.int32)
    pool = Pool(qa, counted(tables, 8), tables)
    assert check(qa, pool, [1], [20], [60])[1] == 0          # three copies and a page: four are free
    pool = Pool(qa, counted(tables, 7), tables)
    assert check(qa, pool, [1], [20], [60])[1] == 1


def forest(rng, n, stride, n_pages):
    """n table rows, each of them an earlier one's prefix with pages of its own behind; and lengths in pages."""
    ids = rng.permutation(n_pages).astype(np.int32)
    tables, held, at = np.full((n, stride), -1, np.int32), [], 0
    for i in range(n):
        shared = 0
        if i and rng.random() < 0.8:
            parent = int(rng.integers(0, i))
            shared = int(rng.integers(0, held[parent] + 1))
            tables[i, :shared] = tables[parent, :shared]
        own = int(rng.integers(0, min(stride - shared, 3) + 1))
        tables[i, shared:shared + own] = ids[at:at + own]
        at += own
        held.append(shared + own)
    return tables, held


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("n,stride,most", [(5, 9, 8), (40, 12, 4), (40, 100, 90), (1024, 6, 6)])
def test_random_families(qa, seed, n, stride, most):
    """Families of rows that share prefixes; a part of them, in any order, writes from anywhere on, over up to `most` pages."""
    rng = np.random.default_rng(100 * n + seed)
    page, n_pages = 16, 3 * n + n * min(most, stride) // 2 + 50
    tables, held = forest(rng, n, stride, n_pages)
    pool = Pool(qa, counted(tables, n_pages), tables, page=page, layers=1, heads=1)
    rows = rng.permutation(n)[:max(1, n - seed)].tolist()
    past = [int(rng.integers(0, held[r] * page + 1)) for r in rows]
    new = [int(rng.integers(0, max(1, min(most * page, stride * page - p)))) for p in past]
    copies, missing = check(qa, pool, rows, past, new)
    assert n < 40 or missing > 0 or len(copies) > 0


def test_more_copies_than_list_entries(qa):
    """One row of a pair writes over 1500 pages that both hold."""
    n = 1500
    tables = np.tile(np.random.default_rng(1).permutation(2 * n + 7)[:n].astype(np.int32), (2, 1))
    pool = Pool(qa, counted(tables, 2 * n + 7), tables, layers=1, heads=1)
    copies, _ = check(qa, pool, [0], [3], [16 * n])
    assert len(copies) == n


def test_captured_extends_replay(qa):
    """Replays of one graph, eager calls in between, on lengths that the host changes: steps that copy nothing, one page, many."""
    hip = Hip()
    stride, n_pages, page = 30, 200, 16
    tables = np.full((4, stride), -1, np.int32)
    tables[:, :20] = np.random.default_rng(2).permutation(n_pages)[:20]
    host = ref.pool_of(np.random.default_rng(3), 2, n_pages, 2, page, True)
    lay = ref.layout(qa, 2, n_pages, 2, page, True)
    dev = qa.DeviceArray.from_numpy
    d_pool, d_refs, d_tables = dev(host), dev(counted(tables, n_pages)), dev(tables)
    rows, past, new = dev(np.arange(4, dtype=np.int32)), dev(np.zeros(4, np.int32)), dev(np.zeros(4, np.int32))
    ws_bytes = qa.lib.qa_pages_workspace_bytes(C.byref(lay))
    ws, missing = qa.DeviceArray((ws_bytes,), np.uint8), qa.DeviceArray((1,), np.int32)

    def enqueue(stream):
        qa.check(qa.lib.qa_pages_extend(d_pool.ptr, C.byref(lay), d_refs.ptr, d_tables.ptr, 4, stride, rows.ptr, past.ptr, new.ptr, 4,
                                        missing.ptr, ws.ptr, ws_bytes, stream))

    stream = hip.stream()
    graph, run = hip.capture(stream, lambda: enqueue(stream))
    for turn, (p, n) in enumerate([([310, 250, 200, 5], [1, 1, 90, 300]), ([320, 300, 200, 20], [1, 1, 1, 1]),
                                   ([0, 0, 0, 0], [100, 200, 30, 40]), ([7, 7, 7, 7], [300, 300, 300, 300])] * 2):
        state = counted(tables, n_pages), tables, host
        for again in (0, 1):                                        # from the same state, replayed and eager
            refs, t, copies, lacking = extend(state[0], state[1], page, range(4), p, n)
            moved = state[2].copy()
            for a, b in copies:
                moved[:, :, b] = state[2][:, :, a]
            d_refs.upload(state[0])
            d_tables.upload(state[1])
            d_pool.upload(state[2])
            past.upload(np.array(p, np.int32))
            new.upload(np.array(n, np.int32))
            if again:
                enqueue(None)
            else:
                hip.hipGraphLaunch(run, stream)
            qa.synchronize()
            assert int(missing.numpy()[0]) == lacking
            np.testing.assert_array_equal(d_refs.numpy(), refs)
            np.testing.assert_array_equal(d_tables.numpy(), t)
            np.testing.assert_array_equal(d_pool.numpy().view(np.uint8), moved.view(np.uint8))
        tables, host = t, moved
        if turn == 3:                                               # all share again
            tables = np.tile(tables[3], (4, 1))
    hip.drop(graph, run)
    hip.hipStreamDestroy(stream)
