"""Attention on pages of 8 bits where rows of V differ in size by many powers of two: seen ones, unseen ones, and ones that weigh nothing.

Every column (a token's head) is held against its own sum of p times a row's largest |v|, so that large rows which a token does not
see, or hardly, cannot hide an error of its result.  Tolerance, of that sum: a score of normal q and k is off by at most 2 parts
in 2^22 of |q| |k| scale, which is below 16 here: 2^-17; a probability is off by that and its normaliser by as much; the exponential,
two f16 parts and the sums add a few 2^-22.  2^-16 holds all of it twice over for the sizes that occur (|q| |k| scale about 11, errors of
the 128 products of either sign).  (The parts of p times a row's scale leave out up to 2^-25 where a column's largest is 2^-1 to 2^14, and
that of every dim: where the largest row has a 0, the others' sum is good to the largest row's 2^-24, not to its own.)"""
import numpy as np
import pytest

import candidates_ref as cand
import paged_ref as ref

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -16


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


class Case:
    def __init__(self, qa, past, news, kv_heads=8, group=2, page=16, seed=11):
        self.qa, self.page, self.news = qa, page, news
        self.rng = np.random.default_rng(seed)
        self.tables, pages = ref.tables_of(self.rng, [p + n for p, n in zip(past, news)], page)
        self.pool = cand.Pool(qa, "q8", 1, pages, kv_heads, page, self.rng)
        self.heads = kv_heads * group
        self.b = ref.Batch(qa, self.tables, past, news)
        self.q = self.rng.standard_normal((self.b.rows, self.heads * 128)).astype(np.float32)

    def scale(self, seq, pos, by, kv=1):
        """Multiplies the scales of a position's rows."""
        self.pool.scales[0, kv, self.tables[seq, pos // self.page], :, pos % self.page] *= np.float32(by)

    def check(self, mask=None, workspace=None):
        print(f"q8 scales past={self.b.past.tolist()} news={self.news} tree={mask is not None}", flush=True)
        got = cand.run_attention(self.qa, self.q, self.pool, 0, self.b, self.heads, mask=mask, workspace=workspace).astype(np.float64)
        values = self.pool.values
        size = values.copy()
        size[:, 1] = np.abs(size[:, 1]).max(-1, keepdims=True)
        args = 0, self.tables, self.page, self.b.past, self.b.start, self.heads
        if mask is None:
            want, own = (ref.attention(self.q, v, *args) for v in (values, size))
        else:
            want, own = (cand.tree_attention(self.q, v, *args, mask) for v in (values, size))
        assert np.isfinite(got).all()
        off = np.abs(got - want) / np.where(own > 0, own, 1)
        worst = np.unravel_index(off.argmax(), off.shape)
        assert off.max() <= TOL, (worst, off.max(), got[worst], want[worst], own[worst])


CHUNKS = [([37], [3], 8), ([37], [30], 8), ([5, 300, 0], [1, 70, 20], 8), ([3000], [64], 8), ([1500], [300], 2)]


@pytest.mark.parametrize("past,news,kv_heads", CHUNKS)
@pytest.mark.parametrize("power", [12, 30, 100])
def test_later_tokens_do_not_matter(qa, past, news, kv_heads, power):
    """V of some of the chunk's tokens is 2^power times the others': those before them do not see it."""
    c = Case(qa, past, news, kv_heads)
    for s, (p, n) in enumerate(zip(past, news)):
        for t in sorted({n - 1, n - 1 - n // 5, n // 2} - {0}):
            c.scale(s, p + t, 2.0 ** power)
    c.check()


@pytest.mark.parametrize("past,nodes,kv_heads", [([30], [8], 8), ([156, 300, 20], [20, 41, 1], 8), ([2000, 2000], [32, 32], 8), ([700], [64], 2)])
@pytest.mark.parametrize("power", [12, 30, 100])
def test_siblings_do_not_matter(qa, past, nodes, kv_heads, power):
    c = Case(qa, past, nodes, kv_heads)
    rng = np.random.default_rng(power)
    parents = np.concatenate([cand.random_tree(rng, n) for n in nodes])
    for s, (p, n) in enumerate(zip(past, nodes)):
        for t in range(2, n, 5):
            c.scale(s, p + t, 2.0 ** power)
    mask, _ = cand.masks_of(parents, c.b.start, c.b.rows, 2)
    c.check(mask)


@pytest.mark.parametrize("past,news,kv_heads", [([200], [1], 8), ([3900, 40], [1, 1], 8)] + CHUNKS)
@pytest.mark.parametrize("power", [20, 45])
def test_rows_that_weigh_nothing(qa, past, news, kv_heads, power):
    """A cached key that the first head's tokens answer with a probability of about 2^-65 has V of 2^power times the others'."""
    c = Case(qa, past, news, kv_heads)
    c.q[:] = np.tile(c.q[:1], (c.b.rows, 1))                       # every token asks the same
    for s, p in enumerate(past):
        if p == 0:
            continue
        for pos in (p // 3, p - 1):
            at = 0, 0, c.tables[s, pos // 16], slice(None), pos % 16
            rows = -4 * c.q[0].reshape(kv_heads, -1, 128)[:, 0]
            c.pool.ints[at], c.pool.scales[at] = cand.quantise(rows)
            c.scale(s, pos, 2.0 ** power)
    c.check()


@pytest.mark.parametrize("past,news,kv_heads", [([900], [1], 8), ([12000], [1], 2)] + CHUNKS)
@pytest.mark.parametrize("spread", [16, 60, 110])
def test_any_sizes(qa, past, news, kv_heads, spread):
    """Scales up to 2^spread apart, and rows of zeros: the sums of the probabilities hold their keys whatever V is."""
    c = Case(qa, past, news, kv_heads)
    v = c.pool.scales[:, 1]
    v *= np.exp2(c.rng.integers(-spread // 2, spread // 2 + 1, v.shape)).astype(np.float32)
    v[c.rng.random(v.shape) < 0.3] = 0
    c.check()
    c.check(workspace=0)


@pytest.mark.parametrize("past,news,kv_heads", [([900], [1], 8)] + CHUNKS[1:4])
@pytest.mark.parametrize("power", [-100, -82, 90])
def test_all_rows_small_or_large(qa, past, news, kv_heads, power):
    """All rows of V, and all but the zeros in front."""
    c = Case(qa, past, news, kv_heads)
    c.pool.scales[:, 1] *= np.float32(2.0 ** power)
    c.check()
    for s, (p, n) in enumerate(zip(past, news)):
        for pos in range((p + n) // 2):
            c.scale(s, pos, 0.0)
    c.check()
