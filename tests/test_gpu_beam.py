"""Beam selection and the reordering of the beams' states, against plain 64-bit statements.

Exponentials are f32 (relative error 2^-22 each), everything behind them 64 bits: a logarithm of a sum is off by at most 2^-22,
and a score, whose f32 rounding adds 2^-24 of itself, by 2^-22 + 2^-24 |score|.  Where two candidates' exact scores are
nearer than 2^-21 their order may differ; the inputs below are checked not to have such pairs, or have exact ties, whose order
is by number."""
import numpy as np
import pytest

import candidates_ref as cand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


def run_select(qa, logits, width, scores, done=None, stops=(), stream=None):
    rows, vocab = logits.shape
    groups = rows // width
    need = qa.lib.qa_beam_select_workspace_bytes(groups, width, vocab)
    assert need > 0
    ws = qa.DeviceArray.from_numpy(np.full(need, 0xff, np.uint8))
    d = [qa.DeviceArray.from_numpy(a) for a in (logits.astype(np.float32), np.asarray(scores, np.float32))]
    d_done = None if done is None else qa.DeviceArray.from_numpy(np.asarray(done, np.int32))
    d_stop = qa.DeviceArray.from_numpy(np.asarray(list(stops) or [0], np.int32))
    out = [qa.DeviceArray.from_numpy(np.full(rows, 99, np.int32)) for _ in range(3)]
    out_scores = qa.DeviceArray.from_numpy(np.full(rows, 99, np.float32))
    print(f"beams {rows} x {vocab}, width {width}", flush=True)
    qa.check(qa.lib.qa_beam_select(d[0].ptr, groups, width, vocab, d[1].ptr, d_done.ptr if d_done else None, d_stop.ptr, len(stops),
                                   out[0].ptr, out[1].ptr, out_scores.ptr, out[2].ptr, ws.ptr, need, stream))
    qa.synchronize()
    return out[0].numpy(), out[1].numpy(), out_scores.numpy(), out[2].numpy()


def check(qa, logits, width, scores, done=None, stops=(), ties=False):
    got = run_select(qa, logits, width, scores, done, stops)
    p, t, s, d, gap = cand.select(np.asarray(logits, np.float32), width, np.asarray(scores, np.float32),
                                  np.zeros(len(logits)) if done is None else done, stops)
    assert ties or gap > 2.0 ** -20, gap
    np.testing.assert_array_equal(got[0], p)
    np.testing.assert_array_equal(got[1], t)
    np.testing.assert_array_equal(got[3], d)
    fine = np.isfinite(s)
    assert (got[2][~fine] == -np.inf).all()
    assert (np.abs(got[2][fine] - s[fine]) <= 2.0 ** -22 + 2.0 ** -24 * np.abs(s[fine])).all()


@pytest.mark.parametrize("groups,width,vocab", [(1, 1, 1), (1, 2, 2), (1, 4, 151936), (1, 1, 151936), (3, 5, 1000), (2, 8, 64), (2, 8, 65), (5, 3, 63), (1, 64, 64),
                                                (1, 64, 151936), (2, 32, 4097), (8, 8, 151936), (1, 16, 2049), (40, 2, 513), (1, 17, 151935), (1, 64, 1500)])
def test_select(qa, groups, width, vocab):
    rng = np.random.default_rng(vocab + width)
    rows = groups * width
    logits = rng.standard_normal((rows, vocab)).astype(np.float32) * 3
    scores = -5 * rng.random(rows)
    done = (rng.random(rows) < 0.2).astype(np.int32)
    check(qa, logits, width, scores, done, stops=(0, int(logits[0].argmax()), vocab - 1))


def test_first_step_and_dead_beams(qa):
    """One beam of four counts: the others' scores are -inf or NaN."""
    rng = np.random.default_rng(1)
    row = rng.standard_normal((1, 5000)).astype(np.float32)
    logits = np.repeat(row, 8, 0)
    check(qa, logits, 4, [0, -np.inf, -np.inf, -np.inf, -np.inf, np.nan, -1.5, -np.inf])


@pytest.mark.parametrize("width,vocab", [(4, 40), (8, 8), (8, 300), (64, 64), (64, 700), (33, 9000), (5, 1500)])
def test_one_beam_of_small_vocabularies(qa, width, vocab):
    """One beam counts and its row has fewer blocks of values than there are beams: all its values are looked at."""
    rng = np.random.default_rng(vocab)
    logits = rng.standard_normal((2 * width, vocab)).astype(np.float32) * 2
    scores = np.full(2 * width, -np.inf)
    scores[width // 2], scores[-1] = -0.5, 0
    check(qa, logits, width, scores)
    done = np.zeros(2 * width, np.int32)
    done[0], scores[0] = 1, -1.0
    check(qa, logits, width, scores, done)


def test_fewer_candidates_than_beams(qa):
    """All beams done, no beam that counts, and rows with few values: the rest is done, with -inf."""
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((16, 100)).astype(np.float32)
    scores = -rng.random(16)
    done = np.zeros(16, np.int32)
    done[:4] = 1
    scores[2] = -np.inf
    scores[4:8] = -np.inf
    logits[8:12] = -np.inf
    logits[8, 7], logits[10, 3] = 1.0, 2.0
    logits[12:16] = np.nan
    check(qa, logits, 4, scores, done)


def test_values_that_are_not_numbers(qa):
    """NaN is no candidate and weighs nothing, -inf neither, a row with +inf has none."""
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((6, 3000)).astype(np.float32)
    logits[0, ::2] = np.nan
    logits[1, 5:2900] = -np.inf
    logits[2, 17] = np.inf
    logits[3, 0] = np.nan
    logits[4] = np.nan
    check(qa, logits, 6, -rng.random(6))


@pytest.mark.parametrize("width,vocab", [(4, 151936), (64, 70), (8, 10000), (64, 9000)])
def test_ties(qa, width, vocab):
    """Rows of one value, and rows that are the same: lower beams and lower ids first."""
    logits = np.zeros((2 * width, vocab), np.float32)
    logits[width:] = np.arange(vocab) % 7
    check(qa, logits, width, np.full(2 * width, -1.0), ties=True)
    rng = np.random.default_rng(0)
    same = np.repeat(rng.standard_normal((1, vocab)).astype(np.float32), width, 0)
    check(qa, same, width, np.full(width, -2.0), ties=True)


@pytest.mark.parametrize("order", ["rising", "falling", "waves"])
def test_values_in_order(qa, order):
    """The best values lie next to each other, or where one wave alone looks."""
    v = 65536
    x = np.arange(v, dtype=np.float32) / 4096
    if order == "falling":
        x = x[::-1].copy()
    if order == "waves":   # one 64-lane block of maxima in sixteen holds everything that counts
        x = np.where((np.arange(v) // 64) % 1024 < 64, x + 100, x)
    logits = np.stack([x, x * np.float32(0.999), x * np.float32(1.001), x * np.float32(0.99)])
    check(qa, logits, 4, [0.0, -0.3, -0.1, -0.2], ties=True)
    check(qa, np.repeat(logits, 16, 0) * (1 + np.arange(64, dtype=np.float32)[:, None] / 1024), 64, -np.arange(64) / 77, ties=True)


def test_large_and_small_scores(qa):
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((4, 4000)).astype(np.float32) * np.float32(1e4)
    check(qa, logits, 4, [-3e4, -1e-30, -2e4, -4e4])
    logits = rng.standard_normal((4, 4000)).astype(np.float32) * np.float32(1e37)
    got = run_select(qa, logits, 4, [0, -1, -2, -3])
    assert got[0].tolist() == [0, 1, 2, 3] and got[1].tolist() == logits.argmax(1).tolist()


def test_rows_past_32_bits(qa):
    """Offsets of the last rows' logits pass 2^31 bytes and 2^29 values."""
    vocab, width = 9000001, 62
    d = qa.DeviceArray((width, vocab), np.float32)          # zeros: 2.2 GB
    need = qa.lib.qa_beam_select_workspace_bytes(1, width, vocab)
    ws = qa.DeviceArray((need,), np.uint8)
    last = np.zeros(vocab, np.float32)
    best = [vocab - 1, 12345, 7000000]
    for k, b in enumerate(best):
        last[b] = 20 - k
    qa.check(qa.lib.qa_copy_to_device(d.ptr.value + 4 * vocab * (width - 1), last.ctypes.data, last.nbytes))
    scores = qa.DeviceArray.from_numpy(np.zeros(width, np.float32))
    out = [qa.DeviceArray((width,), np.int32) for _ in range(3)]
    so = qa.DeviceArray((width,))
    qa.check(qa.lib.qa_beam_select(d.ptr, 1, width, vocab, scores.ptr, None, None, 0, out[0].ptr, out[1].ptr, so.ptr, out[2].ptr, ws.ptr, need, None))
    qa.synchronize()
    assert out[0].numpy()[:3].tolist() == [width - 1] * 3 and out[1].numpy()[:3].tolist() == best
    assert out[0].numpy()[3:].tolist() == [0] * (width - 3) and out[1].numpy()[3:].tolist() == list(range(width - 3))


# ------------------------------------------------------------------------------------------ states
def run_reorder(qa, refs, tables, page, rows, parents, lens, ids=None, tokens=None, ids_len=None, n_rows=None, null_rows=False):
    up = lambda a: None if a is None else qa.DeviceArray.from_numpy(np.asarray(a, np.int32))
    d = [up(a) for a in (refs, tables, None if null_rows else rows, parents, lens, ids, tokens, ids_len)]
    p = [x.ptr if x is not None else None for x in d]
    n_rows = len(tables if tables is not None else ids) if n_rows is None else n_rows
    qa.check(qa.lib.qa_beam_reorder(p[0], 0 if refs is None else len(refs), p[1], n_rows, 0 if tables is None else tables.shape[1], page,
                                    p[2], p[3], p[4], len(parents), p[5], 0 if ids is None else ids.shape[1], p[6], p[7], None))
    qa.synchronize()
    return tuple(None if d[k] is None else d[k].numpy() for k in (0, 1, 5))


def same(got, want):
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        if a is not None:
            np.testing.assert_array_equal(a, b)


def states(rng, n_rows, stride, n_pages, ids_stride):
    tables = rng.integers(0, n_pages, (n_rows, stride)).astype(np.int32)
    tables[rng.random(tables.shape) < 0.2] = -1
    refs = np.bincount(tables[tables >= 0], minlength=n_pages).astype(np.int32)
    return refs, tables, rng.integers(0, 1000, (n_rows, ids_stride)).astype(np.int32)


@pytest.mark.parametrize("n,n_rows,stride,ids_stride,page", [(1, 1, 1, 1, 16), (4, 6, 13, 49, 16), (8, 8, 160, 209, 16), (64, 70, 33, 5, 64), (1024, 1100, 9, 17, 32),
                                                             (300, 300, 260, 1, 256)])
def test_reorder(qa, n, n_rows, stride, ids_stride, page):
    rng = np.random.default_rng(n)
    refs, tables, ids = states(rng, n_rows, stride, 5 * stride, ids_stride)
    rows = rng.permutation(n_rows)[:n].astype(np.int32)
    parents = rng.integers(0, n, n).astype(np.int32)
    lens = rng.integers(0, stride * page + 20, n).astype(np.int32)
    tokens, at = rng.integers(-1, 500, n).astype(np.int32), rng.integers(-1, ids_stride + 1, n).astype(np.int32)
    got = run_reorder(qa, refs, tables, page, rows, parents, lens, ids, tokens, at)
    want = cand.reorder(refs, tables, page, rows, parents, lens, ids, tokens, at)
    same(got, want)
    t = want[1]
    np.testing.assert_array_equal(want[0], np.bincount(t[t >= 0], minlength=len(refs)))
    same(run_reorder(qa, refs, tables, page, rows, parents, lens), cand.reorder(refs, tables, page, rows, parents, lens))
    same(run_reorder(qa, None, None, page, rows, parents, None, ids), cand.reorder(None, None, page, rows, parents, None, ids))
    same(run_reorder(qa, None, None, page, rows, parents, None, ids, tokens, at), cand.reorder(None, None, page, rows, parents, None, ids, tokens, at))


def test_reorder_of_lists_that_are_none(qa):
    """Rows outside the table or listed twice, parents outside the list or among those: such entries keep their rows."""
    rng = np.random.default_rng(9)
    refs, tables, ids = states(rng, 9, 40, 300, 30)
    tables[3, 5], tables[2, 7] = 300, -9                   # numbers of no page
    refs = np.bincount(tables[(tables >= 0) & (tables < 300)], minlength=300).astype(np.int32)
    rows = np.array([3, 8, 3, -1, 9, 2, 5], np.int32)
    parents = np.array([1, 0, 1, 0, 0, 4, 7], np.int32)
    lens = np.array([100, -3, 100, 100, 100, 100, 100], np.int32)
    same(run_reorder(qa, refs, tables, 16, rows, parents, lens, ids), cand.reorder(refs, tables, 16, rows, parents, lens, ids))
    parents = np.array([2, 5, 1, 0, 0, 5, -1], np.int32)
    same(run_reorder(qa, refs, tables, 16, rows, parents, lens, ids), cand.reorder(refs, tables, 16, rows, parents, lens, ids))
    order = np.array([2, 0, 1], np.int32)
    same(run_reorder(qa, refs, tables, 16, None, order, lens[:3] * 0 + 600, ids, null_rows=True),
         cand.reorder(refs, tables, 16, [0, 1, 2], order, [600] * 3, ids))
