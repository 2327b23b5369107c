"""Plain 64-bit statements of the 8-bit cache, of drafted trees and of beam selection, and the buffers of their tests.

A pool of any cache type is a Pool: its values [layer][K, V][page][KV head][position][dim] in 64 bits, and the bytes that the
library gets.  Nothing here is shared with the library."""
import ctypes as C

import numpy as np

import paged_ref as ref

DIM = ref.DIM
CACHES = ("f32", "f16", "q8")


def cache_type(qa, cache):
    return {"f32": qa.QA_CACHE_F32, "f16": qa.QA_CACHE_F16, "q8": qa.QA_CACHE_Q8}[cache]


def quantise(x):
    """(int8 values, f32 scales) of rows [..][128] of f32, as the header says."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        scale = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32)
        q = np.where(scale[..., None] > 0, np.rint(x / scale[..., None]), 0).astype(np.float64)
    bad = ~np.isfinite(x).all(-1)
    q = np.where(bad[..., None], 0, np.clip(q, -127, 127))
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), scale)


class Pool:
    def __init__(self, qa, cache, layers, pages, heads, page, rng=None, values=None):
        self.qa, self.cache, self.page = qa, cache, page
        self.layout = qa.KvLayout(layers, pages, heads, DIM, page, cache_type(qa, cache))
        shape = (layers, 2, pages, heads, page, DIM)
        if values is None:
            values = rng.standard_normal(shape).astype(np.float32) if rng is not None else np.zeros(shape, np.float32)
        if cache == "q8":
            self.ints, self.scales = quantise(values)
        else:
            self.raw = np.ascontiguousarray(values.astype(np.float16 if cache == "f16" else np.float32))

    @property
    def values(self):
        if self.cache != "q8":
            return self.raw.astype(np.float64)
        with np.errstate(invalid="ignore"):
            return self.ints.astype(np.float64) * self.scales.astype(np.float64)[..., None]

    def bytes(self):
        if self.cache != "q8":
            return self.raw.view(np.uint8).reshape(-1)
        head = self.ints.shape[:3]
        return np.concatenate([self.ints.reshape(*head, -1).view(np.uint8),
                               np.ascontiguousarray(self.scales).reshape(*head, -1).view(np.uint8)], -1).reshape(-1)

    def take(self, data):
        """Another pool of the same layout from the library's bytes."""
        out = Pool.__new__(Pool)
        out.qa, out.cache, out.page, out.layout = self.qa, self.cache, self.page, self.layout
        if self.cache != "q8":
            out.raw = data.view(self.raw.dtype).reshape(self.raw.shape)
            return out
        blocks = data.reshape(*self.ints.shape[:3], -1)
        rows = self.ints.shape[3] * self.page
        out.ints = np.ascontiguousarray(blocks[..., :rows * DIM]).view(np.int8).reshape(self.ints.shape)
        out.scales = np.ascontiguousarray(blocks[..., rows * DIM:]).view(np.float32).reshape(self.scales.shape)
        return out

    def upload(self):
        data = self.bytes()
        assert data.size == self.qa.lib.qa_kv_cache_bytes(C.byref(self.layout))
        return self.qa.DeviceArray.from_numpy(data)


def run_attention(qa, q, pool, layer, batch, n_heads, mask=None, scale=ref.SCALE, fill=0.0, workspace=None, stream=None):
    lay = C.byref(pool.layout)
    need = qa.lib.qa_paged_attn_workspace_bytes(lay, batch.ref, n_heads)
    size = need if workspace is None else workspace
    ws = qa.DeviceArray.from_numpy(np.full(max(size, 16), 0xff, np.uint8))      # stale contents: NaN
    d_q, d_pool = qa.DeviceArray.from_numpy(q), pool.upload()
    out = qa.DeviceArray.from_numpy(np.full((q.shape[0], n_heads * DIM), fill, np.float32))
    space = (ws.ptr if size else None, size, stream)
    if mask is None:
        qa.check(qa.lib.qa_paged_attn(d_q.ptr, d_pool.ptr, lay, layer, batch.ref, n_heads, scale, out.ptr, *space))
    else:
        d_mask = qa.DeviceArray.from_numpy(np.ascontiguousarray(mask, np.uint32).view(np.int32))
        qa.check(qa.lib.qa_paged_tree_attn(d_q.ptr, d_pool.ptr, lay, layer, batch.ref, d_mask.ptr, mask.shape[1], n_heads, scale,
                                           out.ptr, *space))
    qa.synchronize()
    return out.numpy().reshape(-1, n_heads, DIM)


# ---- trees
def random_tree(rng, n, reach=5, roots=0.0):
    """Parents of n nodes: one of the `reach` before, -1 for node 0 and for some others."""
    return np.array([-1 if i == 0 or rng.random() < roots else int(rng.integers(max(0, i - reach), i)) for i in range(n)], np.int32)


def ancestors(parents):
    """Per node the list of its ancestors and itself."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def masks_of(parents, start, rows, words):
    """(mask [rows][words], depth [rows]) of the sequences' trees; other rows are zeros."""
    mask, depth = np.zeros((rows, words), np.uint32), np.zeros(rows, np.int32)
    for s in range(len(start) - 1):
        for i, nodes in enumerate(ancestors(parents[start[s]:start[s + 1]])):
            depth[start[s] + i] = len(nodes) - 1
            for j in nodes:
                if j < 32 * words:
                    mask[start[s] + i, j // 32] |= np.uint32(1 << (j % 32))
    return mask, depth


def tree_attention(q, values, layer, tables, page, past, start, n_heads, mask, scale=ref.SCALE, out=None):
    heads, pages = values.shape[3], values.shape[2]
    group = n_heads // heads
    q = q.reshape(-1, n_heads, DIM).astype(np.float64)
    out = np.zeros_like(q) if out is None else out.reshape(q.shape).astype(np.float64)
    for s in range(len(past)):
        n = start[s + 1] - start[s]
        for r in range(start[s], start[s + 1]):
            seen = list(range(past[s])) + [past[s] + i for i in range(min(n, 32 * mask.shape[1])) if mask[r, i // 32] >> np.uint32(i % 32) & 1]
            places = [(int(tables[s, j // page]), j % page) for j in seen if j // page < tables.shape[1]]
            places = [(p, x) for p, x in places if 0 <= p < pages]
            if not places:
                out[r] = 0.0
                continue
            pg, sl = np.array(places).T
            for h in range(n_heads):
                with np.errstate(all="ignore"):
                    x = (values[layer, 0, pg, h // group, sl] @ q[r, h]) * scale
                    e = np.exp(x - x.max())
                    out[r, h] = (e / e.sum()) @ values[layer, 1, pg, h // group, sl]
    return out


def accept(parents, ids, picks):
    """(path, next) of one tree."""
    path, at = [0], 0
    while True:
        child = [i for i in range(at + 1, len(parents)) if parents[i] == at and ids[i] == picks[at]]
        if not child:
            return path, int(picks[at])
        at = child[0]
        path.append(at)


# ---- beams
def select(logits, width, scores, done, stops):
    """(parents, tokens, scores, done, gap): gap is the smallest distance between neighbouring scores up to the first that is left out."""
    rows, vocab = logits.shape
    out, gap = [], np.inf
    for first in range(0, rows, width):
        found = []
        for r in range(first, first + width):
            score = float(scores[r])
            if not np.isfinite(score):
                continue
            if done[r]:
                found.append((-score, r, -1))
                continue
            x = logits[r].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            m = x.max()
            if not np.isfinite(m):
                continue
            v = score + (x - (m + np.log(np.exp(x - m).sum())))
            for i in np.lexsort((np.arange(vocab), -v))[:width + 1]:
                if np.isfinite(v[i]):
                    found.append((-v[i], r, int(i)))
        found.sort()
        for a, b in zip(found[:width], found[1:width + 1]):
            if a[1:] != b[1:] and b[0] > a[0]:
                gap = min(gap, b[0] - a[0])
        for k in range(width):
            if k < len(found):
                s, r, t = found[k]
                out.append((r, t, -s, int(t < 0 or t in stops)))
            else:
                out.append((first + k, -1, -np.inf, 1))
    p, t, s, d = zip(*out)
    return np.array(p, np.int32), np.array(t, np.int32), np.array(s), np.array(d, np.int32), gap


def reorder(refs, tables, page, rows, parents, lens, ids=None, tokens=None, ids_len=None):
    refs, tables = (None, None) if refs is None else (refs.copy(), tables.copy())
    ids = None if ids is None else ids.copy()
    n_rows = len(tables if tables is not None else ids)
    usable, seen = [], set()
    for r in rows:
        usable.append(0 <= r < n_rows and r not in seen)
        seen.add(r)
    before = None if tables is None else tables.copy()
    ids_before = None if ids is None else ids.copy()
    for i, row in enumerate(rows):
        p = parents[i]
        if not usable[i] or not 0 <= p < len(rows) or not usable[p]:
            continue
        if tables is not None:
            for j in range(tables.shape[1]):
                now = int(before[rows[p], j]) if j < -(-max(lens[i], 0) // page) else -1
                now = now if 0 <= now < len(refs) else -1
                old = int(before[row, j])
                tables[row, j] = now
                if now >= 0:
                    refs[now] += 1
                if 0 <= old < len(refs):
                    refs[old] -= 1
        if ids is not None:
            ids[row] = ids_before[rows[p]]
            if tokens is not None and tokens[i] >= 0 and 0 <= ids_len[i] < ids.shape[1]:
                ids[row, ids_len[i]] = tokens[i]
    return refs, tables, ids
