"""Beam selection where the numbers that decide are far smaller than a row's logarithm of its sum, or than a beam's score.

Scores there are rounded in 64 bits at the size of the larger number, and values that lie nearer than that are ties, which go to the
lower id.  Rows of tiny logits differ from each other by 1e-16 of a score and less, so the statement below compares as 64 bits do: a
row's value is raised by one 64-bit number, which is good to 2^-22.  Rows of one group are therefore the same in their
logarithm (the same set of values, in another order), or far apart."""
import numpy as np
import pytest

from test_gpu_beam import run_select

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


def one_row(x, count):
    """The ids of a row's best values, ties to the lower id."""
    return np.lexsort((np.arange(len(x)), -x))[:count].tolist()


@pytest.mark.parametrize("vocab", [700, 20000, 151936])
@pytest.mark.parametrize("size", [1e-6, 1e-9, 1e-12, 1e-30])
@pytest.mark.parametrize("width", [1, 2, 4])
def test_tiny_logits(qa, vocab, size, width):
    """Of each group the last beam alone counts: its best values, in order, whatever its score is.  Values that 64 bits cannot tell
    apart beside the logarithm of the vocabulary may come in the order of their ids."""
    rng = np.random.default_rng(vocab + width)
    groups = 24
    logits = (rng.standard_normal((groups * width, vocab)) * size).astype(np.float32)
    scores = np.full(groups * width, -np.inf)
    scores[width - 1::width] = -50 * rng.random(groups)
    parents, tokens, out, done = run_select(qa, logits, width, scores)
    assert (done == 0).all()
    for g in range(groups):
        row = g * width + width - 1
        x, score = logits[row].astype(np.float64), np.float64(np.float32(scores[row]))
        lse = np.log(np.exp(x - x.max()).sum()) + x.max()
        mine = slice(g * width, (g + 1) * width)
        assert (parents[mine] == row).all() and len(set(tokens[mine])) == width
        # what one addition at the size of the score and the logarithm may round away, once in the value and once in the one it replaces
        off = 2 * np.spacing(abs(score) + abs(lse) + 1)
        np.testing.assert_array_less(np.sort(x)[::-1][:width] - off, x[tokens[mine]] + 1e-300)
        assert (np.abs(out[mine] - (score - lse + x[tokens[mine]])) <= 2.0 ** -22 + 2.0 ** -24 * abs(score - lse)).all()
        order = one_row(x, min(width + 1, vocab))
        if (-np.diff(x[order]) > 2 * off).all():
            assert tokens[mine].tolist() == order[:width]


@pytest.mark.parametrize("peak", [-1e-9, -1.1920929e-7, 1e-9])
@pytest.mark.parametrize("score", [-60.0, -1000.0, -1e10])
def test_sure_tokens_behind_low_scores(qa, peak, score):
    """Log-probabilities of beams that are nearly sure of their token: each beam's one token wins, and the beams keep their order."""
    rng = np.random.default_rng(3)
    groups, width, vocab = 50, 2, 3000
    rows = groups * width
    logits = (-40 - 5 * rng.random((rows, vocab))).astype(np.float32)
    best = rng.integers(0, vocab, rows)
    logits[np.arange(rows), best] = peak
    scores = np.tile([score, score * 1.001], groups) * (1 + 0.001 * np.repeat(rng.random(groups), width))
    parents, tokens, out, done = run_select(qa, logits, width, scores)
    if score > -1e9:
        np.testing.assert_array_equal(parents, np.arange(rows))
        np.testing.assert_array_equal(tokens, best)
    else:
        # the second beam is 1e7 behind: both come from the first, whose other ids lie 40 lower
        assert (parents == np.repeat(np.arange(groups) * width, width)).all()
        np.testing.assert_array_equal(tokens[::2], best[::2])
    assert (done == 0).all()


@pytest.mark.parametrize("score", [-1e10, -1e30, -3.0e38])
@pytest.mark.parametrize("width,vocab", [(1, 5000), (3, 5000), (4, 40000), (8, 600)])
def test_scores_that_hide_the_logits(qa, score, width, vocab):
    """Beams whose score is a mask's lowest value, all logits negative: with -1e10 the logits count to 2e-6, behind -1e30 all are ties and the
    lowest ids come first.  The rows of a group have few candidates in the others, so that such a beam has to give some."""
    rng = np.random.default_rng(width)
    groups = 6
    logits = np.full((groups * width, vocab), -np.inf, np.float32)
    scores = np.full(groups * width, -1.0)
    for g in range(groups):
        last = g * width + width - 1
        logits[last] = -1 - 3 * rng.random(vocab).astype(np.float32)
        scores[last] = score
        for r in range(g * width, last):                       # one candidate in every second beam
            if (r - g * width) % 2 == 0:
                logits[r, rng.integers(0, vocab)] = -2.0
    parents, tokens, out, done = run_select(qa, logits, width, scores)
    assert (done == 0).all()
    for g in range(groups):
        last, first = g * width + width - 1, g * width
        sure = [r for r in range(first, last) if np.isfinite(logits[r]).any()]
        assert sorted(parents[first:first + len(sure)]) == sure
        rest = slice(first + len(sure), first + width)
        assert (parents[rest] == last).all()
        if abs(score) > 1e20:
            assert tokens[rest].tolist() == list(range(width - len(sure)))
        else:
            x = logits[last].astype(np.float64)
            np.testing.assert_array_less(np.sort(x)[::-1][:width - len(sure)] - 4 * np.spacing(abs(score)), x[tokens[rest]])
            assert len(set(tokens[rest])) == width - len(sure)
