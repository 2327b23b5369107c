"""The paged-cache and 4-bit operators together, as a server uses them, and under what servers do to them: graphs that are
captured and replayed, several streams, batches of every kind in one launch.

Tolerances: attention as in test_gpu_paged.py (relative 2-norm 5e-6); 4-bit projections 2e-6 as in test_gpu_gemv_q4.py; a
layer run of both passes its errors through one more projection and the softmax's derivative (at most 1), so the sum of
its parts, 2e-5, bounds it.  f16 cache rows are compared through the reference's own f16 rounding of the same f32 value: a
value next to a tie may round the other way, half a step 2^-11 of one element of a key or row of 128, far below the bars."""
import ctypes as C
import ctypes.util

import numpy as np
import pytest

import paged_ref as ref
import test_gpu_gemv_q4 as q4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(qa):
    assert qa.device_count() > 0, "no HIP device: GPU tests need the MI355X"


class Hip:
    """The HIP runtime that the library has loaded, for streams and graphs."""

    def __init__(self):
        self.lib = C.CDLL("libamdhip64.so.7")

    def __getattr__(self, name):
        f = getattr(self.lib, name)

        def call(*args):
            rc = f(*args)
            assert rc == 0, (name, rc)
        return call

    def stream(self):
        s = C.c_void_p()
        self.hipStreamCreateWithFlags(C.byref(s), 1)      # non-blocking, default priority
        return s

    def capture(self, stream, body):
        """An executable graph of what body() enqueues on the stream."""
        graph, run = C.c_void_p(), C.c_void_p()
        self.hipStreamBeginCapture(stream, 2)             # relaxed: other threads may allocate
        try:
            body()
        finally:
            self.hipStreamEndCapture(stream, C.byref(graph))
        self.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0))
        return graph, run

    def drop(self, graph, run):
        self.hipGraphExecDestroy(run)
        self.hipGraphDestroy(graph)


@pytest.fixture(scope="module")
def hip(_gpu):
    return Hip()


class Server:
    """Sequences in pages with their host mirror: the K and V that each one has appended, in 64 bits."""

    HEADS, KV = 16, 8

    def __init__(self, qa, rows, stride, pages, page, f16, seed=0):
        self.qa, self.page, self.f16, self.n_pages = qa, page, f16, pages
        self.rng = np.random.default_rng(seed)
        self.lay = ref.layout(qa, 2, pages, self.KV, page, f16)
        dt = np.float16 if f16 else np.float32
        self.dt = dt
        self.pool = qa.DeviceArray.from_numpy(np.full((2, 2, pages, self.KV, page, 128), np.nan, dt))   # nothing may be read
        self.refs = qa.DeviceArray((pages,), np.int32)
        self.tables = qa.DeviceArray.from_numpy(np.full((rows, stride), -1, np.int32))
        self.shape = (rows, stride)
        self.ws = qa.DeviceArray((qa.lib.qa_pages_workspace_bytes(C.byref(self.lay)),), np.uint8)
        self.missing = qa.DeviceArray((1,), np.int32)
        self.k = [np.zeros((0, self.KV, 128)) for _ in range(rows)]
        self.v = [np.zeros((0, self.KV, 128)) for _ in range(rows)]
        self.qn, self.kn = ((1 + 0.1 * self.rng.standard_normal(128)).astype(np.float32) for _ in range(2))
        self.d_qn, self.d_kn = qa.DeviceArray.from_numpy(self.qn), qa.DeviceArray.from_numpy(self.kn)
        self.keep = []

    def ints(self, v):
        self.keep.append(self.qa.DeviceArray.from_numpy(np.asarray(v, np.int32)))
        return self.keep[-1].ptr

    def step(self, news, stream=None):
        """New tokens for the rows of `news` (row: tokens) at once; checks every output."""
        qa, lib = self.qa, self.qa.lib
        rows = sorted(news)
        past = [len(self.k[r]) for r in rows]
        new = [news[r] for r in rows]
        qa.check(lib.qa_pages_extend(self.pool.ptr, C.byref(self.lay), self.refs.ptr, self.tables.ptr, *self.shape, self.ints(rows),
                                     self.ints(past), self.ints(new), len(rows), self.missing.ptr, self.ws.ptr, self.ws.nbytes, stream))
        qa.synchronize()
        assert self.missing.numpy()[0] == 0
        # the batch is the whole table: rows without new tokens are idle sequences
        all_new = [news.get(r, 0) for r in range(self.shape[0])]
        all_past = [len(k) for k in self.k]
        start = np.concatenate([[0], np.cumsum(all_new)]).astype(np.int32)
        n = int(start[-1])
        batch = qa.PagedBatch(self.tables.ptr, self.ints(all_past), self.ints(start), *self.shape, n, max(all_new),
                              max(p + t for p, t in zip(all_past, all_new)))
        qkv = self.rng.standard_normal((n, 4096)).astype(np.float32)
        d_qkv, d_q, out = qa.DeviceArray.from_numpy(qkv), qa.DeviceArray((n, 2048)), qa.DeviceArray((n, 2048))
        need = lib.qa_paged_attn_workspace_bytes(C.byref(self.lay), C.byref(batch), 16)
        ws = qa.DeviceArray((max(need, 16),), np.uint8)
        print(f"step past={all_past} new={all_new} page={self.page} f16={self.f16}", flush=True)
        qa.check(lib.qa_paged_append(d_qkv.ptr, self.d_qn.ptr, self.d_kn.ptr, d_q.ptr, self.pool.ptr, C.byref(self.lay), 1,
                                     C.byref(batch), 16, 1e6, 1e-6, stream))
        qa.check(lib.qa_paged_attn(d_q.ptr, self.pool.ptr, C.byref(self.lay), 1, C.byref(batch), 16, ref.SCALE, out.ptr, ws.ptr,
                                   need, stream))
        qa.synchronize()
        got, q = out.numpy().reshape(n, 16, 128), d_q.numpy().reshape(n, 16, 128)
        worst = 0.0
        for r in rows:
            x = qkv[start[r]:start[r + 1]].reshape(-1, 32, 128)
            pos = np.arange(len(x)) + all_past[r]
            k = np.stack([ref.rope_norm(a[16:24], self.kn, p) for a, p in zip(x, pos)])
            self.k[r] = np.concatenate([self.k[r], k.astype(np.float32).astype(self.dt).astype(np.float64)])
            self.v[r] = np.concatenate([self.v[r], x[:, 24:].astype(self.dt).astype(np.float64)])
            for i, p in enumerate(pos):
                wq = ref.rope_norm(x[i, :16], self.qn, p)
                assert np.abs(q[start[r] + i] - wq).max() <= 2.0 ** -20 * np.abs(wq).max()
                want = self.attend(q[start[r] + i].astype(np.float64), r, p)
                worst = max(worst, np.linalg.norm(got[start[r] + i] - want) / np.linalg.norm(want))
        # K rows of the reference are rounded from 64-bit values, the cache's from f32: a tie now and then, 2^-11 of one
        # value in 128 of one key, weighted by its probability
        assert worst <= (2e-5 if not self.f16 else 1e-4), worst

    def attend(self, q, r, p):
        out = np.zeros((16, 128))
        for h in range(16):
            s = self.k[r][:p + 1, h // 2] @ q[h] * ref.SCALE
            e = np.exp(s - s.max())
            out[h] = (e / e.sum()) @ self.v[r][:p + 1, h // 2]
        return out

    def fork(self, src, dst, n):
        self.qa.check(self.qa.lib.qa_pages_fork(self.refs.ptr, self.n_pages, self.tables.ptr, *self.shape, self.page, self.ints([src]),
                                                self.ints([dst]), self.ints([n]), 1, None))
        self.k[dst], self.v[dst] = self.k[src][:n].copy(), self.v[src][:n].copy()

    def free(self, r, n=0):
        self.qa.check(self.qa.lib.qa_pages_free(self.refs.ptr, self.n_pages, self.tables.ptr, *self.shape, self.page, self.ints([r]),
                                                self.ints([n]), 1, None))
        self.k[r], self.v[r] = self.k[r][:n], self.v[r][:n]

    def compact(self):
        live = self.qa.DeviceArray((1,), np.int32)
        self.qa.check(self.qa.lib.qa_pages_compact(self.pool.ptr, C.byref(self.lay), self.refs.ptr, self.tables.ptr, *self.shape,
                                                   self.refs.ptr, self.tables.ptr, live.ptr, self.ws.ptr, self.ws.nbytes, None))
        self.qa.synchronize()
        n = int(live.numpy()[0])
        assert (self.refs.numpy()[n:] <= 0).all() and (self.refs.numpy()[:n] > 0).all()
        return n


@pytest.mark.parametrize("f16,page", [(True, 16), (False, 32), (True, 128)])
def test_a_served_conversation(qa, f16, page):
    """Prompts in chunks beside streams that generate, beams forked and written apart, a stream that ends, a pool that is
    compacted and serves on.  Pages hold NaN until they are written, and what is freed is given out again."""
    s = Server(qa, rows=6, stride=8 if page > 64 else 24, pages=40 if page < 64 else 16, page=page, f16=f16)
    s.step({0: 100})                         # a prompt
    s.step({0: 1, 2: 37})                    # a token beside another prompt
    s.step({0: 1, 2: 70, 4: 5})              # a chunk, a token, a short one
    s.fork(0, 1, 102)
    s.fork(0, 3, 90)                         # a beam that goes back twelve tokens
    s.step({0: 1, 1: 1, 2: 1, 3: 1, 4: 1})   # three holders of a page write at once
    s.step({1: 1, 3: 20, 5: 16})
    s.free(2)
    s.free(0, 50)
    n = s.compact()
    s.step({0: 3, 1: 1, 2: 18, 3: 1, 4: 40, 5: 1})
    assert s.compact() >= n


def test_the_paged_step_agrees_with_the_contiguous_one(qa):
    """One decode step of three streams over the same K and V in both layouts: the contiguous kernel rounds q and the
    probabilities to f16, so the two agree to its own bar (2e-3, 1e-3)."""
    rng = np.random.default_rng(9)
    lens = [40, 700, 1]
    flat_lay = ref.layout(qa, 1, 3, 8, 1024, True)
    flat = np.zeros((1, 2, 3, 8, 1024, 128), np.float16)
    tables, pages = ref.tables_of(rng, [n + 1 for n in lens], 64)
    pool = np.zeros((1, 2, pages, 8, 64, 128), np.float16)
    for s, n in enumerate(lens):
        rows = rng.standard_normal((2, 8, n, 128)).astype(np.float16)
        flat[0, :, s, :, :n] = rows
        for j in range(n):
            pool[0, :, tables[s, j // 64], :, j % 64] = rows[:, :, j]
    qkv = (rng.standard_normal((3, 4096))).astype(np.float32)
    w = np.ones(128, np.float32)
    d_flat, d_pool, d_qkv, d_w = (qa.DeviceArray.from_numpy(a) for a in (flat, pool, qkv, w))
    d_past = qa.DeviceArray.from_numpy(np.array(lens, np.int32))
    nb = qa.lib.qa_decode_attn_workspace_bytes(3, 16, 1024)
    ws, out = qa.DeviceArray((nb,), np.uint8), qa.DeviceArray((3, 2048))
    qa.check(qa.lib.qa_decode_step_attn(d_qkv.ptr, d_w.ptr, d_w.ptr, d_flat.ptr, C.byref(flat_lay), 0, d_past.ptr, 3, 701, 16, 1e6, 1e-6,
                                        ref.SCALE, out.ptr, ws.ptr, nb, None))
    lay = ref.layout(qa, 1, pages, 8, 64, True)
    b = ref.Batch(qa, tables, lens, [1, 1, 1])
    q, got = qa.DeviceArray((3, 2048)), qa.DeviceArray((3, 2048))
    qa.check(qa.lib.qa_paged_append(d_qkv.ptr, d_w.ptr, d_w.ptr, q.ptr, d_pool.ptr, C.byref(lay), 0, b.ref, 16, 1e6, 1e-6, None))
    qa.check(qa.lib.qa_paged_attn(q.ptr, d_pool.ptr, C.byref(lay), 0, b.ref, 16, ref.SCALE, got.ptr, None, 0, None))
    qa.synchronize()
    a, p = out.numpy(), got.numpy()
    assert np.abs(a - p).max() <= 2e-3 and np.linalg.norm(a - p) <= 1e-3 * np.linalg.norm(p)
    cache = d_pool.numpy()
    for s, n in enumerate(lens):                       # and both appended the same bits
        np.testing.assert_array_equal(cache[0, :, tables[s, n // 64], :, n % 64], d_flat.numpy()[0, :, s, :, n])


class Layer:
    """Projection, append, attention and output projection of one layer's step on 4-bit weights; its buffers."""

    def __init__(self, qa, past, news, f16, seed):
        rng = np.random.default_rng(seed)
        self.qa, self.f16 = qa, f16
        self.hidden = 256
        self.tables, self.pages = ref.tables_of(rng, [p + n for p, n in zip(past, news)], 32)
        self.host = ref.pool_of(rng, 1, self.pages, 8, 32, f16)
        self.batch = ref.Batch(qa, self.tables, past, news)
        n = self.batch.rows
        self.rows = n
        self.w = {"qkv": q4.weights(rng, 4096, self.hidden, 64), "o": q4.weights(rng, self.hidden, 2048, 32)}
        self.x = rng.standard_normal((n, self.hidden)).astype(np.float32)
        self.norm = (1 + 0.1 * rng.standard_normal(self.hidden)).astype(np.float32)
        dev = qa.DeviceArray.from_numpy
        self.pool, self.d_x, self.d_norm, self.d_one = dev(self.host), dev(self.x), dev(self.norm), dev(np.ones(128, np.float32))
        self.d_w = {k: tuple(dev(a) for a in q4.packed(*v)) for k, v in self.w.items()}
        self.qkv, self.q, self.att, self.y = (qa.DeviceArray((n, m)) for m in (4096, 2048, 2048, self.hidden))
        self.lay = ref.layout(qa, 1, self.pages, 8, 32, f16)
        self.need = qa.lib.qa_paged_attn_workspace_bytes(C.byref(self.lay), self.batch.ref, 16)
        self.ws = qa.DeviceArray((max(self.need, 16),), np.uint8)

    def enqueue(self, stream):
        qa, lib, lay = self.qa, self.qa.lib, C.byref(self.lay)
        for r0 in range(0, self.rows, 32):                # 32 rows per projection
            n = min(32, self.rows - r0)
            at = lambda d, width: C.c_void_p(d.ptr.value + r0 * width * 4)  # noqa: E731
            qa.check(lib.qa_gemv_q4(self.d_w["qkv"][0].ptr, self.d_w["qkv"][1].ptr, 64, 4096, self.hidden, at(self.d_x, self.hidden), n,
                                    at(self.qkv, 4096), 0, self.d_norm.ptr, 1e-6, stream))
        qa.check(lib.qa_paged_append(self.qkv.ptr, self.d_one.ptr, self.d_one.ptr, self.q.ptr, self.pool.ptr, lay, 0, self.batch.ref, 16, 1e6,
                                     1e-6, stream))
        qa.check(lib.qa_paged_attn(self.q.ptr, self.pool.ptr, lay, 0, self.batch.ref, 16, ref.SCALE, self.att.ptr, self.ws.ptr, self.need, stream))
        for r0 in range(0, self.rows, 32):
            n = min(32, self.rows - r0)
            at = lambda d, width: C.c_void_p(d.ptr.value + r0 * width * 4)  # noqa: E731
            qa.check(lib.qa_gemv_q4(self.d_w["o"][0].ptr, self.d_w["o"][1].ptr, 32, self.hidden, 2048, at(self.att, 2048), n,
                                    at(self.y, self.hidden), 0, None, 1e-6, stream))

    def want(self):
        """The layer from its own device q and cache rows on: projections and attention in 64 bits."""
        qkv, _ = q4.plain(*self.w["qkv"], self.x, 0, self.norm)
        pool = self.pool.numpy()
        att = ref.attention(self.q.numpy(), pool, 0, self.tables, 32, self.batch.past, self.batch.start, 16)
        y, _ = q4.plain(*self.w["o"], att.reshape(self.rows, 2048).astype(np.float32), 0)
        return qkv, att, y

    def check(self):
        qkv, att, y = self.want()
        for got, want in ((self.qkv.numpy(), qkv), (self.att.numpy().reshape(att.shape), att), (self.y.numpy(), y)):
            assert np.isfinite(got).all()
            assert np.linalg.norm(got - want) <= 2e-5 * np.linalg.norm(want)

    def clear(self):
        for d in (self.qkv, self.q, self.att, self.y):
            d.upload(np.full(d.shape, np.nan, np.float32))
        self.pool.upload(self.host)


BATCHES = [([200, 13, 0], [1, 1, 1]), ([900, 40, 3], [1, 20, 3]), ([300, 0, 64], [1, 100, 70])]


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past,news", BATCHES)
def test_layer_on_4_bit_weights(qa, f16, past, news):
    layer = Layer(qa, past, news, f16, 3)
    layer.enqueue(None)
    qa.synchronize()
    layer.check()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("past,news", BATCHES)
def test_captured_layer_replays(qa, hip, f16, past, news):
    """Replays of a captured step give the eager step's bits every time, with eager work and new inputs in between."""
    layer = Layer(qa, past, news, f16, 5)
    stream = hip.stream()
    graph, run = hip.capture(stream, lambda: layer.enqueue(stream))
    for turn in range(4):
        layer.x = (np.random.default_rng(turn).standard_normal(layer.x.shape)).astype(np.float32)
        layer.d_x.upload(layer.x)
        layer.clear()
        layer.enqueue(None)                               # eager, on the null stream
        qa.synchronize()
        eager = [d.numpy() for d in (layer.qkv, layer.q, layer.att, layer.y, layer.pool)]
        layer.clear()
        hip.hipGraphLaunch(run, stream)
        qa.synchronize()
        for a, d in zip(eager, (layer.qkv, layer.q, layer.att, layer.y, layer.pool)):
            np.testing.assert_array_equal(a.view(np.uint8), d.numpy().view(np.uint8))
        layer.check()
    hip.drop(graph, run)
    hip.hipStreamDestroy(stream)


def test_captured_page_bookkeeping_replays(qa, hip):
    """free, fork, extend and compact of a beam step as one graph, whose lengths the host changes between the replays."""
    stride, pages, page = 12, 60, 16
    lay = ref.layout(qa, 2, pages, 2, page, True)
    rng = np.random.default_rng(0)
    tables = np.full((4, stride), -1, np.int32)
    tables[0, :7] = rng.permutation(pages)[:7]
    refs = np.zeros(pages, np.int32)
    refs[tables[0, :7]] = 1
    host = ref.pool_of(rng, 2, pages, 2, page, True)
    dev = qa.DeviceArray.from_numpy
    d_pool, d_refs, d_tables = dev(host), dev(refs), dev(tables)
    rows, src = dev(np.array([1, 2, 3], np.int32)), dev(np.zeros(3, np.int32))
    lens, new = dev(np.zeros(3, np.int32)), dev(np.array([1, 20, 3], np.int32))
    ws_bytes = qa.lib.qa_pages_workspace_bytes(C.byref(lay))
    ws, missing, live = qa.DeviceArray((ws_bytes,), np.uint8), qa.DeviceArray((1,), np.int32), qa.DeviceArray((1,), np.int32)

    def enqueue(stream):
        t = (d_refs.ptr, pages, d_tables.ptr, 4, stride, page)
        qa.check(qa.lib.qa_pages_free(*t, rows.ptr, None, 3, stream))
        qa.check(qa.lib.qa_pages_fork(*t, src.ptr, rows.ptr, lens.ptr, 3, stream))
        qa.check(qa.lib.qa_pages_extend(d_pool.ptr, C.byref(lay), d_refs.ptr, d_tables.ptr, 4, stride, rows.ptr, lens.ptr, new.ptr, 3,
                                        missing.ptr, ws.ptr, ws_bytes, stream))
        qa.check(qa.lib.qa_pages_compact(d_pool.ptr, C.byref(lay), d_refs.ptr, d_tables.ptr, 4, stride, d_refs.ptr, d_tables.ptr, live.ptr,
                                         ws.ptr, ws_bytes, stream))

    stream = hip.stream()
    graph, run = hip.capture(stream, lambda: enqueue(stream))
    for turn, n in enumerate([100, 112, 33, 1, 100]):
        lens.upload(np.full(3, n, np.int32))
        refs, tables = ref.free(refs, tables, page, [1, 2, 3], [0, 0, 0])
        refs, tables = ref.fork(refs, tables, page, [0, 0, 0], [1, 2, 3], [n] * 3)
        refs, tables, copies, lacking = ref.extend(refs, tables, page, [1, 2, 3], [n] * 3, [1, 20, 3])
        old = host.copy()
        for a, b in copies:
            host[:, :, b] = old[:, :, a]
        refs, tables, moves, count = ref.compact(refs, tables)
        old = host.copy()
        for a, b in moves:
            host[:, :, b] = old[:, :, a]
        if turn % 2:
            enqueue(None)
        else:
            hip.hipGraphLaunch(run, stream)
        qa.synchronize()
        assert (int(missing.numpy()[0]), int(live.numpy()[0])) == (lacking, count) == (0, count)
        np.testing.assert_array_equal(d_refs.numpy(), refs)
        np.testing.assert_array_equal(d_tables.numpy(), tables)
        np.testing.assert_array_equal(d_pool.numpy().view(np.uint8), host.view(np.uint8))
    hip.drop(graph, run)
    hip.hipStreamDestroy(stream)


def test_steps_on_several_streams(qa, hip):
    """Four layers of their own buffers on four streams at once: nothing is shared behind the caller's back."""
    layers = [Layer(qa, past, news, f16, 20 + i) for i, ((past, news), f16) in enumerate(zip(BATCHES + BATCHES[1:2], (True, False, True, True)))]
    streams = [hip.stream() for _ in layers]
    for turn in range(3):
        for layer in layers:
            layer.clear()
        qa.synchronize()
        for _ in range(4):
            for layer, stream in zip(layers, streams):
                layer.enqueue(stream)
        qa.synchronize()
        for layer in layers:
            layer.check()
    for stream in streams:
        hip.hipStreamDestroy(stream)
