"""Plain 64-bit statements of the paged-cache operators, and the buffers of their tests.

A pool is numpy [layer][K, V][page][KV head][position][dim], tables and counts int32.  Nothing here is shared with the
library: rows, pages and positions are walked one by one."""
import ctypes as C

import numpy as np

DIM = 128
SCALE = 1.0 / np.sqrt(128.0)


def layout(qa, layers, pages, heads, page, f16):
    return qa.KvLayout(layers, pages, heads, DIM, page, qa.QA_CACHE_F16 if f16 else qa.QA_CACHE_F32)


def pool_of(rng, layers, pages, heads, page, f16):
    return rng.standard_normal((layers, 2, pages, heads, page, DIM)).astype(np.float16 if f16 else np.float32)


def tables_of(rng, lengths, page, extra=1, spare=3):
    """Table rows of the pages that the lengths need, in random order, and the pool's page count."""
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    ids = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lengths), max(counts + [1]) + extra), -1, np.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = ids[at:at + c]
        at += c
    return table, pages


def visible(table, pages, page, pos):
    """(page, slot) of every position up to pos that lies on a page."""
    out = []
    for j in range(min(pos + 1, len(table) * page)):
        p = int(table[j // page])
        if 0 <= p < pages:
            out.append((p, j % page))
    return out


def attention(q, pool, layer, tables, page, past, start, n_heads, scale=SCALE, out=None):
    """out [rows][n_heads][128] in 64 bits; rows of no sequence keep what `out` holds."""
    heads = pool.shape[3]
    group = n_heads // heads
    q = q.reshape(-1, n_heads, DIM).astype(np.float64)
    out = np.zeros_like(q) if out is None else out.reshape(q.shape).astype(np.float64)
    for s in range(len(past)):
        places = None
        for r in range(start[s], min(start[s + 1], len(q))):
            pos = int(past[s]) + r - int(start[s])
            places = visible(tables[s], pool.shape[2], page, pos)
            if not places:
                out[r] = 0.0
                continue
            pg, sl = np.array(places).T
            for h in range(n_heads):
                k = pool[layer, 0, pg, h // group, sl].astype(np.float64)
                v = pool[layer, 1, pg, h // group, sl].astype(np.float64)
                with np.errstate(all="ignore"):
                    x = (k @ q[r, h]) * scale
                    e = np.exp(x - x.max())
                    out[r, h] = (e / e.sum()) @ v
    return out


class Batch:
    """Device buffers of a ragged batch."""

    def __init__(self, qa, tables, past, news, n_rows=None, max_tokens=None, max_len=None):
        self.start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.past = np.asarray(past, np.int32)
        self.rows = int(self.start[-1]) if n_rows is None else n_rows
        self.d = [qa.DeviceArray.from_numpy(np.ascontiguousarray(a)) for a in (tables.astype(np.int32), self.past, self.start)]
        self.struct = qa.PagedBatch(self.d[0].ptr, self.d[1].ptr, self.d[2].ptr, tables.shape[0], tables.shape[1], self.rows,
                                    max(news) if max_tokens is None else max_tokens,
                                    max(p + n for p, n in zip(past, news)) if max_len is None else max_len)
        self.ref = C.byref(self.struct)


def run_attention(qa, q, pool, layer, batch, page, n_heads, scale=SCALE, fill=0.0, workspace=None, stream=None):
    f16 = pool.dtype == np.float16
    lay = layout(qa, pool.shape[0], pool.shape[2], pool.shape[3], page, f16)
    need = qa.lib.qa_paged_attn_workspace_bytes(C.byref(lay), batch.ref, n_heads)
    size = need if workspace is None else workspace
    ws = qa.DeviceArray((max(size, 16),), np.uint8)
    ws.upload(np.full(max(size, 16), 0xff, np.uint8))   # stale contents: NaN
    d_q, d_pool = qa.DeviceArray.from_numpy(q), qa.DeviceArray.from_numpy(pool)
    out = qa.DeviceArray.from_numpy(np.full((q.shape[0], n_heads * DIM), fill, np.float32))
    qa.check(qa.lib.qa_paged_attn(d_q.ptr, d_pool.ptr, C.byref(lay), layer, batch.ref, n_heads, scale, out.ptr,
                                  ws.ptr if size else None, size, stream))
    qa.synchronize()
    return out.numpy().reshape(-1, n_heads, DIM)


def rope_norm(x, w, pos, theta=1.0e6, eps=1e-6):
    """RMSNorm and NEOX rotation of head rows in 64 bits."""
    x = np.asarray(x, np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    a = pos * float(np.float32(theta)) ** (-np.arange(0, DIM, 2) / DIM)
    lo, hi = x[..., :64], x[..., 64:]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], -1)


# ---- bookkeeping of pages, one list entry after another
def valid(p, n):
    return 0 <= p < n


def extend(refs, tables, page, rows, past, new):
    """(refs, tables, copies [(src, dst)], missing) of qa_pages_extend."""
    refs, tables = refs.copy(), tables.copy()
    n_pages, stride = len(refs), tables.shape[1]
    old_refs, old_tables = refs.copy(), tables.copy()
    free = [p for p in range(n_pages) if refs[p] <= 0]
    copies, seen, need = [], set(), 0
    for row, n_past, n_new in zip(rows, past, new):
        if not 0 <= row < len(tables) or n_new <= 0 or n_past < 0:
            continue
        if row in seen:
            continue
        seen.add(row)
        first, last = n_past // page, min(stride, -(-(n_past + n_new) // page))
        for j in range(first, last):
            p = tables[row, j]
            shared = j == first and valid(p, n_pages) and refs[p] > 1
            if valid(p, n_pages) and not shared:
                continue
            need += 1
            if need > len(free):
                continue
            fresh = free[need - 1]
            if shared:
                copies.append((int(p), fresh))
                refs[p] -= 1
            tables[row, j] = fresh
            refs[fresh] = 1
    if need > len(free):
        return old_refs, old_tables, [], need - len(free)
    return refs, tables, copies, 0


def fork(refs, tables, page, src, dst, length):
    refs, tables = refs.copy(), tables.copy()
    n_pages = len(refs)
    before = tables.copy()
    for i, (a, b, n) in enumerate(zip(src, dst, length)):
        if b in list(dst[i + 1:]) or b in list(src) or not 0 <= a < len(tables) or not 0 <= b < len(tables):
            continue
        for j in range(tables.shape[1]):
            p = before[a, j] if j < -(-max(n, 0) // page) else -1
            if valid(before[b, j], n_pages):
                refs[before[b, j]] -= 1
            tables[b, j] = p if valid(p, n_pages) else -1
            if valid(p, n_pages):
                refs[p] += 1
    return refs, tables


def free(refs, tables, page, rows, keep):
    refs, tables = refs.copy(), tables.copy()
    for row, n in zip(rows, keep):
        if not 0 <= row < len(tables):
            continue
        for j in range(-(-max(n, 0) // page), tables.shape[1]):
            if valid(tables[row, j], len(refs)):
                refs[tables[row, j]] -= 1
            tables[row, j] = -1
    return refs, tables


def compact(refs, tables):
    """(refs, tables, moves, n_live)."""
    live = [p for p in range(len(refs)) if refs[p] > 0]
    holes = [p for p in range(len(live)) if refs[p] <= 0]
    movers = [p for p in live if p >= len(live)]
    assert len(holes) == len(movers)
    place = {p: p for p in live}
    out = refs.copy()
    for m, h in zip(movers, holes):
        place[m] = h
        out[h], out[m] = refs[m], 0
    new = np.array([[place.get(int(p), -1) for p in row] for row in tables], np.int32).reshape(tables.shape)
    return out, new, list(zip(movers, holes)), len(live)
