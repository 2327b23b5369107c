"""Drafted trees, beams and caches of every type together, as a server uses them, and under what servers do to them: graphs that
are captured and replayed, two streams at once, caches past 32 bits.

Tolerances: attention 5e-6 in the 2-norm, as in the operators' own tests, twice where two such results are compared with each
other; rows that are moved or appended a second time are compared bit by bit."""
import ctypes as C

import numpy as np
import pytest

import candidates_ref as cand
import paged_ref as ref
from test_gpu_paged_serving import Hip

pytestmark = pytest.mark.gpu

VOCAB = 40


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


@pytest.fixture(scope="module")
def hip(_gpu):
    return Hip()


class Cache:
    """A pool of which nothing may be read that was not written (bytes 0xff: NaN), its tables and counts."""

    def __init__(self, qa, cache, rows, stride, pages, page, layers=2):
        self.qa, self.page, self.cache = qa, page, cache
        self.shape, self.pages = (rows, stride), pages
        self.layout = qa.KvLayout(layers, pages, 8, 128, page, cand.cache_type(qa, cache))
        self.lay = C.byref(self.layout)
        self.pool = qa.DeviceArray.from_numpy(np.full(qa.lib.qa_kv_cache_bytes(self.lay), 0xff, np.uint8))
        self.refs, self.missing = qa.DeviceArray((pages,), np.int32), qa.DeviceArray((1,), np.int32)
        self.tables = qa.DeviceArray.from_numpy(np.full((rows, stride), -1, np.int32))
        self.ws = qa.DeviceArray((qa.lib.qa_pages_workspace_bytes(self.lay),), np.uint8)
        self.held = []

    def ints(self, v):
        self.held.append(self.qa.DeviceArray.from_numpy(np.asarray(v, np.int32)))
        return self.held[-1].ptr

    def extend(self, past, new):
        n = len(past)
        self.qa.check(self.qa.lib.qa_pages_extend(self.pool.ptr, self.lay, self.refs.ptr, self.tables.ptr, *self.shape, None, self.ints(past),
                                                  self.ints(new), n, self.missing.ptr, self.ws.ptr, self.ws.nbytes, None))
        self.qa.synchronize()
        assert int(self.missing.numpy()[0]) == 0

    def batch(self, past, new):
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        b = self.qa.PagedBatch(self.tables.ptr, self.ints(past), self.ints(start), *self.shape, int(start[-1]), int(max(new)),
                               int(max(p + n for p, n in zip(past, new))))
        return b, start

    def read(self, lengths):
        """The K and V of the first positions of every sequence, f32, one after another."""
        b, start = self.batch([0] * len(lengths), lengths)
        k, v = (self.qa.DeviceArray((max(1, int(start[-1])), 8, 128)) for _ in range(2))
        out = []
        for layer in range(self.layout.n_layers):
            self.qa.check(self.qa.lib.qa_paged_read(self.pool.ptr, self.lay, layer, C.byref(b), k.ptr, v.ptr, self.qa.QA_CACHE_F32, None))
            self.qa.synchronize()
            out.append((k.numpy()[:start[-1]], v.numpy()[:start[-1]]))
        return out


class Model:
    """Token ids to projection rows, and an id to the one that it picks."""

    def __init__(self, qa, seed=0):
        rng = np.random.default_rng(seed)
        self.rows = rng.standard_normal((2, VOCAB, 4096)).astype(np.float32)
        self.norms = [qa.DeviceArray.from_numpy((1 + 0.1 * rng.standard_normal(128)).astype(np.float32)) for _ in range(2)]

    def pick(self, ids):
        return (7 * np.asarray(ids) + 3) % VOCAB


def layers(qa, model, cache, ids, past, new, depth=None, mask=None):
    """Appends the ids' rows and attends in both layers; [layer][rows][16][128]."""
    b, start = cache.batch(past, new)
    n = int(start[-1])
    q, out = qa.DeviceArray((n, 2048)), qa.DeviceArray((n, 2048))
    need = qa.lib.qa_paged_attn_workspace_bytes(cache.lay, C.byref(b), 16)
    ws = qa.DeviceArray.from_numpy(np.full(max(need, 16), 0xff, np.uint8))
    got = []
    for layer in range(2):
        qkv = qa.DeviceArray.from_numpy(model.rows[layer][ids])
        args = (qkv.ptr, model.norms[0].ptr, model.norms[1].ptr, q.ptr, cache.pool.ptr, cache.lay, layer, C.byref(b))
        if depth is None:
            qa.check(qa.lib.qa_paged_append(*args, 16, 1e6, 1e-6, None))
            qa.check(qa.lib.qa_paged_attn(q.ptr, cache.pool.ptr, cache.lay, layer, C.byref(b), 16, ref.SCALE, out.ptr, ws.ptr, need, None))
        else:
            qa.check(qa.lib.qa_paged_tree_append(*args, depth.ptr, 16, 1e6, 1e-6, None))
            qa.check(qa.lib.qa_paged_tree_attn(q.ptr, cache.pool.ptr, cache.lay, layer, C.byref(b), mask.ptr, mask.shape[1], 16, ref.SCALE,
                                               out.ptr, ws.ptr, need, None))
        qa.synchronize()
        got.append(out.numpy().reshape(n, 16, 128))
    return got


@pytest.mark.parametrize("cache", cand.CACHES)
@pytest.mark.parametrize("page", [16, 64])
def test_drafting(qa, cache, page):
    """Steps of drafted trees leave the cache, and give the outputs, that the accepted tokens one after another do."""
    rng = np.random.default_rng(page)
    model = Model(qa)
    drafted, plain = (Cache(qa, cache, 4, 12, 40, page) for _ in range(2))
    prompts = [20, 1, 47, 3]
    text = [rng.integers(0, VOCAB, n).tolist() for n in prompts]
    ids = np.concatenate(text)
    for c in (drafted, plain):
        c.extend([0] * 4, prompts)
        layers(qa, model, c, ids, [0] * 4, prompts)
    first = [int(model.pick(t[-1])) for t in text]           # certain, not yet in the cache
    kept_most = 0
    for step in range(6):
        past = [len(t) for t in text]
        sizes = [int(rng.integers(1, 34)) if step else 1 for _ in text]
        parents = [cand.random_tree(rng, n, 4) for n in sizes]
        fed = []
        for s, p in enumerate(parents):
            x = np.zeros(len(p), np.int32)
            x[0] = first[s]
            for i in range(1, len(p)):
                x[i] = model.pick(x[p[i]]) if rng.random() < 0.6 else rng.integers(0, VOCAB)
            fed.append(x)
        fed = np.concatenate(fed)
        drafted.extend(past, sizes)
        b, start = drafted.batch(past, sizes)
        n = int(start[-1])
        words = -(-max(sizes) // 32)
        d_par, d_ids = qa.DeviceArray.from_numpy(np.concatenate(parents)), qa.DeviceArray.from_numpy(fed)
        mask, depth, path = qa.DeviceArray((n, words), np.int32), qa.DeviceArray((n,), np.int32), qa.DeviceArray((n,), np.int32)
        kept, nxt = qa.DeviceArray((4,), np.int32), qa.DeviceArray((4,), np.int32)
        picks = qa.DeviceArray.from_numpy(model.pick(fed).astype(np.int32))
        qa.check(qa.lib.qa_tree_prepare(C.byref(b), d_par.ptr, mask.ptr, words, depth.ptr, None))
        got = layers(qa, model, drafted, fed, past, sizes, depth, mask)
        qa.check(qa.lib.qa_tree_accept(C.byref(b), d_par.ptr, d_ids.ptr, picks.ptr, path.ptr, kept.ptr, nxt.ptr, None))
        qa.check(qa.lib.qa_paged_keep(drafted.pool.ptr, drafted.lay, C.byref(b), path.ptr, kept.ptr, None))
        qa.synchronize()
        n_kept, paths = kept.numpy().tolist(), path.numpy()
        rows = [start[s] + paths[start[s]:start[s] + n_kept[s]] for s in range(4)]
        new = [fed[r].tolist() for r in rows]
        for s in range(4):
            want, last = cand.accept(parents[s], fed[start[s]:start[s + 1]], model.pick(fed[start[s]:start[s + 1]]))
            assert (rows[s] - start[s]).tolist() == want and int(nxt.numpy()[s]) == last
        # the same tokens in a row
        plain.extend(past, n_kept)
        again = layers(qa, model, plain, np.concatenate(new), past, n_kept)
        at = 0
        for s in range(4):
            for layer in range(2):
                a, c = got[layer][rows[s]].astype(np.float64), again[layer][at:at + n_kept[s]]
                assert np.linalg.norm(a - c) <= 1e-5 * np.linalg.norm(c)
            at += n_kept[s]
            text[s] += new[s]
        first = nxt.numpy().tolist()
        kept_most = max(kept_most, *n_kept)
        lengths = [len(t) for t in text]
        for x, y in zip(drafted.read(lengths), plain.read(lengths)):
            for i in (0, 1):
                assert np.isfinite(x[i]).all()
                np.testing.assert_array_equal(x[i], y[i])
    assert kept_most >= 4


@pytest.mark.parametrize("cache", cand.CACHES)
def test_beam_search(qa, cache):
    """Beams of two utterances over several steps: what each beam's table holds is what its ids say, and the search is the host's."""
    rng = np.random.default_rng(7)
    model = Model(qa, 3)
    groups, width, steps, stops = 2, 4, 14, (5, 11)
    n = groups * width
    c = Cache(qa, cache, n, 6, 60, 16)
    prompts = [19, 30]
    text = [rng.integers(0, VOCAB, p).tolist() for p in prompts for _ in range(width)]
    for g in range(groups):
        for b in range(1, width):
            text[g * width + b] = list(text[g * width])
    # the first beam of each group appends the prompt, the others share it
    past, new = [0] * n, [prompts[r // width] if r % width == 0 else 0 for r in range(n)]
    c.extend(past, new)
    layers(qa, model, c, np.concatenate([text[0], text[width]]), past, new)
    others = [r for r in range(n) if r % width]
    lib = qa.lib
    qa.check(lib.qa_pages_fork(c.refs.ptr, c.pages, c.tables.ptr, *c.shape, 16, c.ints([r - r % width for r in others]), c.ints(others),
                               c.ints([prompts[r // width] for r in others]), len(others), None))
    ids = qa.DeviceArray.from_numpy(np.full((n, steps + 2), -9, np.int32))
    scores, done = qa.DeviceArray((n,)), qa.DeviceArray((n,), np.int32)
    scores.upload(np.array([0.0 if r % width == 0 else -np.inf for r in range(n)], np.float32))
    parents, tokens = qa.DeviceArray((n,), np.int32), qa.DeviceArray((n,), np.int32)
    next_scores, next_done = qa.DeviceArray((n,)), qa.DeviceArray((n,), np.int32)
    need = lib.qa_beam_select_workspace_bytes(groups, width, VOCAB)
    ws = qa.DeviceArray((need,), np.uint8)
    d_stops = qa.DeviceArray.from_numpy(np.array(stops, np.int32))
    out_ids = [[] for _ in range(n)]
    for step in range(steps):
        logits = np.stack([np.random.default_rng([g // width, step] + out_ids[g]).standard_normal(VOCAB) * 2 for g in range(n)]).astype(np.float32)
        d_logits = qa.DeviceArray.from_numpy(logits)
        was = scores.numpy(), done.numpy()
        qa.check(lib.qa_beam_select(d_logits.ptr, groups, width, VOCAB, scores.ptr, done.ptr, d_stops.ptr, len(stops), parents.ptr, tokens.ptr,
                                    next_scores.ptr, next_done.ptr, ws.ptr, need, None))
        lens = [len(t) for t in text]
        qa.check(lib.qa_beam_reorder(c.refs.ptr, c.pages, c.tables.ptr, *c.shape, 16, None, parents.ptr,
                                     c.ints([lens[p] for p in range(n)]) if step == 0 else c.ints(lens_of(parents, lens, qa)), n, ids.ptr,
                                     steps + 2, tokens.ptr, c.ints([len(out_ids[p]) for p in range(n)]) if step == 0 else
                                     c.ints(lens_of(parents, [len(o) for o in out_ids], qa)), None))
        qa.synchronize()
        p, t, s, d, gap = cand.select(logits, width, was[0], was[1], stops)
        assert gap > 2.0 ** -20
        assert parents.numpy().tolist() == p.tolist() and tokens.numpy().tolist() == t.tolist() and next_done.numpy().tolist() == d.tolist()
        text = [text[q] + ([int(x)] if x >= 0 else []) for q, x in zip(p, t)]
        out_ids = [out_ids[q] + ([int(x)] if x >= 0 else []) for q, x in zip(p, t)]
        scores, next_scores = next_scores, scores
        done, next_done = next_done, done
        # the new token's rows, for beams that go on
        new = [1 if x >= 0 else 0 for x in t]
        past = [len(x) - w for x, w in zip(text, new)]
        c.extend(past, new)
        if sum(new):
            layers(qa, model, c, np.array([x[-1] for x, w in zip(text, new) if w]), past, new)
        tables, refs = c.tables.numpy(), c.refs.numpy()
        np.testing.assert_array_equal(refs, np.bincount(tables[tables >= 0], minlength=c.pages))
        got = ids.numpy()
        for r in range(n):
            assert got[r, :len(out_ids[r])].tolist() == out_ids[r]
        lengths = [len(x) for x in text]
        for layer, (k, v) in enumerate(c.read(lengths)):
            at = 0
            for x in text:
                want = model.rows[layer][x].reshape(-1, 32, 128)[:, 24:]
                if cache == "q8":
                    i, sc = cand.quantise(want)
                    want = i.astype(np.float32) * sc[..., None]
                elif cache == "f16":
                    want = want.astype(np.float16).astype(np.float32)
                np.testing.assert_array_equal(v[at:at + len(x)], want)
                at += len(x)
    assert done.numpy().any()


def lens_of(parents, lens, qa):
    qa.synchronize()
    return [lens[p] for p in parents.numpy()]


class Step:
    """A drafting step's calls and a beam step's, on buffers of their own."""

    def __init__(self, qa, cache, past, news, seed, page=16):
        rng = np.random.default_rng(seed)
        self.qa = qa
        tables, pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], page)
        self.start_pool = cand.Pool(qa, cache, 2, pages, 8, page, rng).bytes()
        self.layout = qa.KvLayout(2, pages, 8, 128, page, cand.cache_type(qa, cache))
        self.b = ref.Batch(qa, tables, past, news)
        n = self.b.rows
        self.words = -(-max(news) // 32)
        up = qa.DeviceArray.from_numpy
        ids = rng.integers(0, 3, n).astype(np.int32)
        self.par, self.ids, self.picks = up(np.concatenate([cand.random_tree(rng, k) for k in news])), up(ids), up(rng.integers(0, 3, n).astype(np.int32))
        self.qkv, self.w = up(rng.standard_normal((n, 4096)).astype(np.float32)), up(np.ones(128, np.float32))
        self.pool = up(self.start_pool)
        zeros = lambda *s, t=np.int32: qa.DeviceArray(s, t)
        self.mask, self.depth, self.path, self.kept, self.next = zeros(n, self.words), zeros(n), zeros(n), zeros(len(news)), zeros(len(news))
        self.q, self.out, self.k, self.v = (zeros(n, d, t=np.float32) for d in (2048, 2048, 1024, 1024))
        self.need = qa.lib.qa_paged_attn_workspace_bytes(C.byref(self.layout), self.b.ref, 16)
        self.ws = zeros(max(self.need, 16), t=np.uint8)
        # beams
        self.logits, self.scores = up(rng.standard_normal((12, 3001)).astype(np.float32)), up(-rng.random(12).astype(np.float32))
        self.done = up((rng.random(12) < 0.2).astype(np.int32))
        self.start_tables = rng.integers(0, 50, (12, 30)).astype(np.int32)
        self.start_ids = rng.integers(0, 99, (12, 21)).astype(np.int32)
        self.tables, self.refs, self.hist = zeros(12, 30), zeros(50), zeros(12, 21)
        self.lens, self.at = up(np.full(12, 400, np.int32)), up(np.full(12, 20, np.int32))
        self.parents, self.tokens, self.ended, self.so = zeros(12), zeros(12), zeros(12), zeros(12, t=np.float32)
        self.bneed = qa.lib.qa_beam_select_workspace_bytes(3, 4, 3001)
        self.bws = zeros(self.bneed, t=np.uint8)
        self.results = [self.mask, self.depth, self.q, self.out, self.path, self.kept, self.next, self.k, self.v, self.pool, self.parents, self.tokens,
                        self.so, self.ended, self.tables, self.refs, self.hist]

    def reset(self):
        for r in self.results:
            r.upload(np.full(r.shape, 77, r.dtype))
        self.pool.upload(self.start_pool)
        self.tables.upload(self.start_tables)
        self.refs.upload(np.bincount(self.start_tables.ravel(), minlength=50).astype(np.int32))
        self.hist.upload(self.start_ids)
        self.ws.upload(np.full(self.ws.shape, 0xff, np.uint8))
        self.bws.upload(np.full(self.bws.shape, 0xff, np.uint8))
        self.qa.synchronize()

    def enqueue(self, stream):
        qa, lib, lay = self.qa, self.qa.lib, C.byref(self.layout)
        qa.check(lib.qa_tree_prepare(self.b.ref, self.par.ptr, self.mask.ptr, self.words, self.depth.ptr, stream))
        qa.check(lib.qa_paged_tree_append(self.qkv.ptr, self.w.ptr, self.w.ptr, self.q.ptr, self.pool.ptr, lay, 1, self.b.ref, self.depth.ptr, 16,
                                          1e6, 1e-6, stream))
        qa.check(lib.qa_paged_tree_attn(self.q.ptr, self.pool.ptr, lay, 1, self.b.ref, self.mask.ptr, self.words, 16, ref.SCALE, self.out.ptr,
                                        self.ws.ptr if self.need else None, self.need, stream))
        qa.check(lib.qa_tree_accept(self.b.ref, self.par.ptr, self.ids.ptr, self.picks.ptr, self.path.ptr, self.kept.ptr, self.next.ptr, stream))
        qa.check(lib.qa_paged_keep(self.pool.ptr, lay, self.b.ref, self.path.ptr, self.kept.ptr, stream))
        qa.check(lib.qa_paged_read(self.pool.ptr, lay, 1, self.b.ref, self.k.ptr, self.v.ptr, qa.QA_CACHE_F32, stream))
        qa.check(lib.qa_beam_select(self.logits.ptr, 3, 4, 3001, self.scores.ptr, self.done.ptr, None, 0, self.parents.ptr, self.tokens.ptr,
                                    self.so.ptr, self.ended.ptr, self.bws.ptr, self.bneed, stream))
        qa.check(lib.qa_beam_reorder(self.refs.ptr, 50, self.tables.ptr, 12, 30, 16, None, self.parents.ptr, self.lens.ptr, 12, self.hist.ptr, 21,
                                     self.tokens.ptr, self.at.ptr, stream))

    def values(self):
        return [r.numpy() for r in self.results]


# trees on one tile with ranges to join, on 32-column tiles of 8 waves, and of few columns beside longer ones
BATCHES = [("q8", [3000], [20]), ("f16", [500 + 20 * i for i in range(16)], [40 - i for i in range(16)]), ("f32", [600, 650], [63, 60]),
           ("q8", [2000] * 3 + [300] * 9, [50] + [2] * 11)]


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_capture_in_every_mode(qa, hip, mode):
    steps = [Step(qa, *b, seed=i) for i, b in enumerate(BATCHES)]
    stream = hip.stream()
    graph, run = C.c_void_p(), C.c_void_p()
    hip.hipStreamBeginCapture(stream, mode)
    try:
        for s in steps:
            s.enqueue(stream)
    finally:
        hip.hipStreamEndCapture(stream, C.byref(graph))
    hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0))
    for _ in range(3):
        eager = []
        for s in steps:
            s.reset()
            s.enqueue(None)
        qa.synchronize()
        for s in steps:
            eager.append(s.values())
            assert np.isfinite(eager[-1][3]).all() and eager[-1][5].max() >= 2
            s.reset()
        hip.hipGraphLaunch(run, stream)
        qa.synchronize()
        for s, want in zip(steps, eager):
            for a, b in zip(s.values(), want):
                np.testing.assert_array_equal(a, b)
    hip.drop(graph, run)
    hip.hipStreamDestroy(stream)


@pytest.mark.parametrize("handle", [None, 1, 2])
def test_default_streams(qa, handle):
    s = Step(qa, *BATCHES[0], seed=3)
    s.reset()
    s.enqueue(None)
    qa.synchronize()
    want = s.values()
    s.reset()
    s.enqueue(C.c_void_p(handle))
    qa.synchronize()
    for a, b in zip(s.values(), want):
        np.testing.assert_array_equal(a, b)


def test_two_streams_at_once(qa, hip):
    steps = [Step(qa, *b, seed=i) for i, b in enumerate(BATCHES)]
    want = []
    for s in steps:
        s.reset()
        s.enqueue(None)
        qa.synchronize()
        want.append(s.values())
        s.reset()
    streams = [hip.stream(), hip.stream()]
    for _ in range(2):
        for i, s in enumerate(steps):
            s.enqueue(streams[i % 2])
        qa.synchronize()
        for s, w in zip(steps, want):
            for a, b in zip(s.values(), w):
                np.testing.assert_array_equal(a, b)
            s.reset()
    for st in streams:
        hip.hipStreamDestroy(st)


def test_8_bits_past_32_bits(qa):
    """Blocks of 17000 pages of 256 positions: K and V lie 4.6 GB apart, rows and scales past 2^32 bytes."""
    pages, page = 17000, 256
    lay = qa.KvLayout(1, pages, 8, 128, page, qa.QA_CACHE_Q8)
    pool = qa.DeviceArray((qa.lib.qa_kv_cache_bytes(C.byref(lay)),), np.uint8, zero=False)
    assert pool.nbytes > 9e9
    tables = np.array([[pages - 1, 3, pages - 2], [16001, pages - 3, -1]], np.int32)
    rng = np.random.default_rng(0)
    past, new = [0, 0], [600, 300]
    b = ref.Batch(qa, tables, past, new)
    qkv = rng.standard_normal((900, 4096)).astype(np.float32)
    d_qkv, w, q = qa.DeviceArray.from_numpy(qkv), qa.DeviceArray.from_numpy(np.ones(128, np.float32)), qa.DeviceArray((900, 2048))
    out, k, v = qa.DeviceArray((900, 2048)), qa.DeviceArray((900, 8, 128)), qa.DeviceArray((900, 8, 128))
    qa.check(qa.lib.qa_paged_append(d_qkv.ptr, w.ptr, w.ptr, q.ptr, pool.ptr, C.byref(lay), 0, b.ref, 16, 1e6, 1e-6, None))
    qa.check(qa.lib.qa_paged_read(pool.ptr, C.byref(lay), 0, b.ref, k.ptr, v.ptr, qa.QA_CACHE_F32, None))
    need = qa.lib.qa_paged_attn_workspace_bytes(C.byref(lay), b.ref, 16)
    ws = qa.DeviceArray((max(16, need),), np.uint8)
    qa.check(qa.lib.qa_paged_attn(q.ptr, pool.ptr, C.byref(lay), 0, b.ref, 16, ref.SCALE, out.ptr, ws.ptr, need, None))
    qa.synchronize()
    i, s = cand.quantise(qkv.reshape(900, 32, 128)[:, 24:])
    values = i.astype(np.float32) * s[..., None]
    np.testing.assert_array_equal(v.numpy(), values)
    kk, got, qq = k.numpy().astype(np.float64), out.numpy().reshape(900, 16, 128), q.numpy().reshape(900, 16, 128).astype(np.float64)
    for r in (0, 255, 256, 300, 511, 512, 599, 600, 855, 856, 899):
        lo = 0 if r < 600 else 600
        for h in (0, 5, 15):
            x = kk[lo:r + 1, h // 2] @ qq[r, h] * ref.SCALE
            e = np.exp(x - x.max())
            want = (e / e.sum()) @ values[lo:r + 1, h // 2].astype(np.float64)
            assert np.linalg.norm(got[r, h] - want) <= 5e-6 * np.linalg.norm(want)
    # 300 rows moved together from the third page of the first sequence
    path = np.full(900, -1, np.int32)
    path[:299] = np.arange(301, 600)
    d_path, kept = qa.DeviceArray.from_numpy(path), qa.DeviceArray.from_numpy(np.array([299, 0], np.int32))
    qa.check(qa.lib.qa_paged_keep(pool.ptr, C.byref(lay), b.ref, d_path.ptr, kept.ptr, None))
    qa.check(qa.lib.qa_paged_read(pool.ptr, C.byref(lay), 0, b.ref, None, v.ptr, qa.QA_CACHE_F32, None))
    qa.synchronize()
    np.testing.assert_array_equal(v.numpy()[:299], values[301:600])
    np.testing.assert_array_equal(v.numpy()[299:], values[299:])
