"""Attention over pages with long chunks: many tokens behind many positions, which the call cuts into larger tiles and key
ranges of their own, alone and beside sequences of one token.  Statements and tolerances are those of the shorter calls
(a relative 2-norm error of 5e-6, a value within 2^-16 of the largest |v|)."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import case, close

pytestmark = pytest.mark.gpu

LAYOUT = dict(kv_heads=2, group=8)   # 200 tokens are 1600 columns of a KV head


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past,news,page", [
    ([1200], [200], 16), ([1999], [129], 256), ([0], [700], 64), ([4075], [33], 32),
    ([1501, 40, 700, 0, 0], [157, 1, 200, 0, 2], 32), ([3, 2500, 900], [1, 1, 260], 16), ([2000, 1000], [100, 100], 128),
])
def test_long_chunks(qa, f16, past, news, page):
    got, want, pool, *_ = case(qa, 100 + past[0], past, news, page, f16, **LAYOUT)
    close(got, want, np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("group,news", [(1, 1400), (3, 470), (5, 300), (16, 80)])
def test_groups(qa, f16, group, news):
    got, want, pool, *_ = case(qa, group, [1500, 31], [news, 1], 32, f16, kv_heads=1, group=group)
    close(got, want, np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("holes", [
    [(0, j, -1) for j in range(0, 40)], [(0, 0, -1), (0, 41, 2 ** 31 - 1), (0, 81, -9)], [(0, j, lambda n: n) for j in range(0, 88, 2)],
    [(0, j, -1) for j in range(0, 88)],
])
def test_positions_without_a_page(qa, f16, holes):
    got, want, pool, *_ = case(qa, 17, [1200, 60], [200, 1], 16, f16, holes=holes, fill=5.0, **LAYOUT)
    close(got, want, np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past", [[1200], [1200, 300]])
def test_any_workspace_and_bounds(qa, f16, past):
    """Without a workspace, with a part of it, with all; without bounds of the host; rows that belong to no sequence."""
    news = [200, 1][:len(past)]
    args = (qa, 41, past, news, 32, f16)
    full, want, pool, *_ = case(*args, **LAYOUT)
    vmax = np.abs(pool.astype(np.float64)).max()
    close(full, want, vmax)
    np.testing.assert_array_equal(full.view(np.uint32), case(*args, **LAYOUT)[0].view(np.uint32))
    rows = sum(news)
    for size in (0, rows * 16 * 130 * 4 * 2 - 16, rows * 16 * 130 * 4 * 3):
        close(case(*args, workspace=size, **LAYOUT)[0], want, vmax)
    got, want, *_ = case(*args, bounds=False, n_rows=rows + 30, fill=7.25, **LAYOUT)
    close(got[:rows], want[:rows], vmax)
    assert (got[rows:] == 7.25).all()


@pytest.mark.parametrize("f16", [True, False])
def test_what_masked_places_hold_does_not_matter(qa, f16):
    rng = np.random.default_rng(3)
    page, past, new = 64, 1301, 210
    tables, pages = ref.tables_of(rng, [past + new], page)
    pool = ref.pool_of(rng, 1, pages, 2, page, f16)
    clean = pool.copy()
    held = np.isin(np.arange(pages), tables[0])
    pool[:, :, ~held] = np.nan
    pool[:, :, tables[0, (past + new - 1) // page], :, (past + new) % page:] = np.inf
    # the last half of the tokens have keys and values that are not finite: the first half sees none of them
    for j in range(past + new // 2, past + new):
        pool[0, j % 2, tables[0, j // page], :, j % page, j % 128] = np.nan if j % 3 else np.inf
    b = ref.Batch(qa, tables, [past], [new])
    q = rng.standard_normal((new, 16 * 128)).astype(np.float32)
    got = ref.run_attention(qa, q, pool, 0, b, page, 16)
    want = ref.attention(q, clean, 0, tables, page, b.past, b.start, 16)
    close(got[:new // 2], want[:new // 2], np.abs(clean.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
def test_not_finite_q_stays_in_its_row(qa, f16):
    rng = np.random.default_rng(12)
    news, past = [190, 1], [1400, 9]
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], 16)
    pool = ref.pool_of(rng, 1, pages, 2, 16, f16)
    b = ref.Batch(qa, tables, past, news)
    q = rng.standard_normal((b.rows, 16, 128)).astype(np.float32)
    q[0, 3, 7], q[77, 4, 0], q[189, 15, 1], q[-1, 9, 100] = np.nan, np.inf, np.nan, -np.inf
    got = ref.run_attention(qa, q.reshape(b.rows, -1), pool, 0, b, 16, 16)
    want = ref.attention(q, pool, 0, tables, 16, b.past, b.start, 16)
    bad = np.isnan(want)
    assert bad[0, 3].all() and bad.sum() >= 3 * 128
    assert np.array_equal(np.isnan(got), bad)
    close(got[~bad], want[~bad], np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
def test_max_len_is_a_hint(qa, f16):
    rng = np.random.default_rng(1)
    past, news = [1400, 2000], [190, 3]
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], 32)
    pool = ref.pool_of(rng, 1, pages, 2, 32, f16)
    q = rng.standard_normal((193, 2048)).astype(np.float32)
    for max_len in (1, 1100, 10 ** 6):
        b = ref.Batch(qa, tables, past, news, max_len=max_len)
        got = ref.run_attention(qa, q, pool, 0, b, 32, 16)
        close(got, ref.attention(q, pool, 0, tables, 32, b.past, b.start, 16), np.abs(pool.astype(np.float64)).max())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("rows", [1023, 1024, 1500])
def test_long_append_gives_the_bits_of_the_contiguous_append(qa, f16, rows):
    """Two sequences of many tokens and one of one, each against its own append; rows of no sequence stay."""
    rng = np.random.default_rng(rows)
    past, news, page = [37, 0, 900], [rows - 420, 417, 1], 64
    qkv = rng.standard_normal((rows, 4096)).astype(np.float32)
    qn, kn = ((1 + 0.1 * rng.standard_normal(128)).astype(np.float32) for _ in range(2))
    tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], page)
    pool = ref.pool_of(rng, 1, pages, 8, page, f16)
    b = ref.Batch(qa, tables, past, news, n_rows=rows)
    d = [qa.DeviceArray.from_numpy(a) for a in (qkv, qn, kn, np.full((rows, 2048), 3.5, np.float32), pool)]
    lay = ref.layout(qa, 1, pages, 8, page, f16)
    print(f"append of {rows} rows f16={f16}", flush=True)
    qa.check(qa.lib.qa_paged_append(*(x.ptr for x in d), C.byref(lay), 0, b.ref, 16, 1e6, 1e-6, None))
    qa.synchronize()
    q, got = d[3].numpy(), d[4].numpy()
    assert (q[sum(news):] == 3.5).all()
    expect = pool.copy()
    flat_lay = ref.layout(qa, 1, 1, 8, 2048, f16)
    for s, (p, n) in enumerate(zip(past, news)):
        r0 = int(b.start[s])
        x = qa.DeviceArray.from_numpy(np.ascontiguousarray(qkv[r0:r0 + n]))
        flat, q0 = qa.DeviceArray((2, 8, 2048, 128), pool.dtype), qa.DeviceArray((n, 2048))
        d_past = qa.DeviceArray.from_numpy(np.array([p], np.int32))
        qa.check(qa.lib.qa_kv_append(x.ptr, d[1].ptr, d[2].ptr, q0.ptr, flat.ptr, C.byref(flat_lay), 0, d_past.ptr, 1, n, 16, 1e6, 1e-6, None))
        qa.synchronize()
        np.testing.assert_array_equal(q0.numpy().view(np.uint32), q[r0:r0 + n].view(np.uint32))
        a = flat.numpy()
        for pos in range(p, p + n):
            expect[0, :, tables[s, pos // page], :, pos % page] = a[:, :, pos]
    np.testing.assert_array_equal(got, expect)
