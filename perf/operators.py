"""Measured workloads of the serving operators: a K/V cache in pages and matrix-vector products with 4-bit weights.

Four kinds of work, on the head shapes of the two released model sizes (16 query heads, 8 KV heads, head_dim 128):

  attn    causal attention of each sequence's new tokens over its pages (one token: a decode step)
  append  RMSNorm and rotary embedding of q and k, and the K/V rows written into the pages
  fork    one beam step of the page bookkeeping: old beams freed, the parent forked, the written page made private
  compact the live pages moved to the lowest places of the pool, tables and counts rewritten
  q4      a projection with 4-bit weights and f16 group scales, for one to 32 token rows

A pool is [layer][k, v][page][KV head][position in the page][dim].  A table row lists the pages of a sequence in
order of position, -1 where there is none; refs counts the table entries that hold a page.
"""
import math
import os
import sys

import torch

own = False

HEADS, KV_HEADS, DIM = 16, 8, 128
GROUP = HEADS // KV_HEADS
Q_DIM, KV_DIM = HEADS * DIM, KV_HEADS * DIM
THETA, EPS = 1.0e6, 1.0e-6
SCALE = 1.0 / math.sqrt(DIM)
# projections of the two model sizes: rows of W, columns of W, whether the rows are gate | up with a SwiGLU behind
MATRICES = {"small_qkv": (4096, 1024, False), "small_head": (151936, 1024, False), "qkv": (4096, 2048, False),
            "o": (2048, 2048, False), "gate_up": (12288, 2048, True), "down": (2048, 6144, False),
            "head": (151936, 2048, False)}


def listed():
    return [
        # One generated token behind an 11 s utterance (156 positions): launches and latency.
        {"name": "attn_token_short", "kind": "attn", "seqs": 1, "shortest": 156, "longest": 156, "chunked": 0,
         "new": 1, "page": 16, "cache": "f16"},
        # A step of 32 served streams, short utterances to five minutes of audio.
        {"name": "attn_streams", "kind": "attn", "seqs": 32, "shortest": 156, "longest": 3913, "chunked": 0,
         "new": 1, "page": 16, "cache": "f16"},
        # A mixed step of a server: three prompts in chunks, nine streams that generate, one token each.
        {"name": "attn_mixed", "kind": "attn", "seqs": 12, "shortest": 24, "longest": 2500, "chunked": 3,
         "new": 250, "page": 64, "cache": "f16"},
        # The last chunk of a five-minute prompt.
        {"name": "attn_chunk_long", "kind": "attn", "seqs": 1, "shortest": 2889, "longest": 2889, "chunked": 1,
         "new": 1024, "page": 32, "cache": "f16"},
        # The drop-in API's default cache type, an utterance behind an earlier one, odd lengths.
        {"name": "attn_chunk_f32", "kind": "attn", "seqs": 2, "shortest": 701, "longest": 1037, "chunked": 2,
         "new": 157, "page": 16, "cache": "f32"},
        # The K/V rows of that step of 32 streams, and of a five-minute prompt.
        {"name": "append_streams", "kind": "append", "seqs": 32, "shortest": 156, "longest": 3913, "chunked": 0,
         "new": 1, "page": 16, "cache": "f16"},
        {"name": "append_prompt", "kind": "append", "seqs": 1, "shortest": 0, "longest": 0, "chunked": 1,
         "new": 3913, "page": 64, "cache": "f16"},
        # Four candidates behind an utterance, and 32 behind five minutes of audio.
        {"name": "fork_few", "kind": "fork", "beams": 4, "prefix": 156, "page": 16, "layers": 28, "cache": "f16"},
        {"name": "fork_many", "kind": "fork", "beams": 32, "prefix": 3913, "page": 16, "layers": 28, "cache": "f16"},
        # A pool of which a third of the pages lies free in between, before it is shrunk.
        {"name": "compact_pool", "kind": "compact", "seqs": 24, "longest": 700, "free": 35, "page": 16, "layers": 28,
         "cache": "f16"},
        # The gate and up projections of one token, and the vocabulary's logits of eight streams.
        {"name": "q4_gate_up_token", "kind": "q4", "matrix": "gate_up", "rows": 1, "group": 32, "norm": True},
        {"name": "q4_head_streams", "kind": "q4", "matrix": "head", "rows": 8, "group": 64, "norm": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "append", "fork", "compact", "q4", "q4"])
    page = rng.choice([16, 32, 64, 128, 256])
    cache = rng.choice(["f16", "f16", "f32"])
    if kind in ("attn", "append"):
        seqs = _log_int(rng, 1, 32)
        a, b = sorted([_log_int(rng, 1, 3913), _log_int(rng, 1, 3913)])
        chunked = rng.choice([0, 0, rng.randrange(1, seqs + 1)])
        # no more new tokens than the largest listed chunk has, fewer where they are many rows' or in f32
        new = min(_log_int(rng, 2, 1024), max(2, (320 if cache == "f32" else 1024) // chunked), 2048 // seqs) if chunked else 1
        a, b = min(a, 3913 - new), min(b, 3913 - new)
        return {"kind": kind, "seqs": seqs, "shortest": a, "longest": b, "chunked": chunked, "new": new, "page": page,
                "cache": cache}
    if kind == "fork":
        return {"kind": kind, "beams": _log_int(rng, 1, 32), "prefix": _log_int(rng, 1, 3913 if page < 64 else 2000),
                "page": page, "layers": 28 if page == 16 else 4, "cache": cache}
    if kind == "compact":
        return {"kind": kind, "seqs": rng.randrange(1, 25), "longest": _log_int(rng, 20, 700),
                "free": rng.randrange(0, 60), "page": page, "layers": 28 if page == 16 else 4,
                "cache": "f16" if page == 16 else cache}
    return {"kind": kind, "matrix": rng.choice(sorted(MATRICES)), "rows": _log_int(rng, 1, 32),
            "group": rng.choice([32, 64, 128]), "norm": rng.choice([True, False])}


# ------------------------------------------------------------------------------------------ what a case is made of
def _pasts(case):
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    return [a + (b - a) * ((7 * i) % n) // max(1, n - 1) if n % 7 else a + (b - a) * i // max(1, n - 1)
            for i in range(n)]


def _news(case):
    """New tokens of each sequence: chunks of falling length first, then one token each."""
    return [max(1, case["new"] - 13 * i) if i < case["chunked"] else 1 for i in range(case["seqs"])]


def _dtype(case):
    return torch.float16 if case["cache"] == "f16" else torch.float32


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(g, counts, stride, pages):
    """Table rows of the given numbers of pages, drawn without order from a pool of `pages`."""
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(counts), stride), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = ids[at:at + c]
        at += c
    return table


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["kind"] in ("attn", "append"):
        past, new, ps = _pasts(case), _news(case), case["page"]
        counts = [-(-(p + n) // ps) for p, n in zip(past, new)]
        rows = sum(new)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        layers, s["layer"] = 2, 1
        pages = sum(counts) + 5
        s["pages"] = _normal(g, layers, 2, pages, KV_HEADS, ps, DIM, dtype=_dtype(case))
        s["tables"] = _tables(g, counts, max(counts) + 1, pages)
        s["n_past"], s["row_start"] = _ints(past), _ints(starts)
        s["rows"], s["max_new"], s["max_len"] = rows, max(new), max(p + n for p, n in zip(past, new))
        if case["kind"] == "attn":
            s["q"] = _normal(g, rows, Q_DIM)
            s["out"] = torch.zeros(rows, Q_DIM, device="cuda")
        else:
            s["qkv"] = _normal(g, rows, Q_DIM + 2 * KV_DIM)
            s["q_norm"], s["k_norm"] = (1.0 + _normal(g, DIM, std=0.1) for _ in range(2))
            s["q"] = torch.zeros(rows, Q_DIM, device="cuda")
    elif case["kind"] == "fork":
        # row 0 is the parent; every beam holds the parent's full pages and two pages of its own
        ps, n, prefix = case["page"], case["beams"], case["prefix"]
        full, parent = prefix // ps, -(-prefix // ps)
        pages, stride = parent + 2 * n + n + 3, parent + 4
        ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        tables = torch.full((n + 1, stride), -1, dtype=torch.int32, device="cuda")
        tables[0, :parent] = ids[:parent]
        tables[1:, :full] = ids[:full]
        tables[1:, full:full + 2] = ids[parent:parent + 2 * n].view(n, 2)
        s["tables"] = tables
        s["refs"] = torch.bincount(tables[tables >= 0], minlength=pages).to(torch.int32)
        s["pages"] = _normal(g, case["layers"], 2, pages, KV_HEADS, ps, DIM, dtype=_dtype(case))
        s["beams"], s["parents"] = _ints(list(range(1, n + 1))), _ints([0] * n)
        s["lens"], s["ones"] = _ints([prefix] * n), _ints([1] * n)
        s["missing"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    elif case["kind"] == "compact":
        ps = case["page"]
        lens = [max(1, case["longest"] - (37 * i) % case["longest"]) for i in range(case["seqs"])]
        counts = [-(-v // ps) for v in lens]
        pages = max(sum(counts) + 1, sum(counts) * 100 // (100 - case["free"]))
        s["tables"] = _tables(g, counts, max(counts) + 2, pages)
        s["refs"] = torch.bincount(s["tables"][s["tables"] >= 0], minlength=pages).to(torch.int32)
        s["pages"] = _normal(g, case["layers"], 2, pages, KV_HEADS, ps, DIM, dtype=_dtype(case))
        s["tables_out"], s["refs_out"] = torch.empty_like(s["tables"]), torch.empty_like(s["refs"])
        s["live"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        n, k, swiglu = MATRICES[case["matrix"]]
        tiles = n // 16
        # 16 rows x 128 columns in 1 KB, and the rows' scales of each group of columns
        s["weights"] = torch.randint(0, 256, (tiles, k // 128, 64, 16), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = (0.002 + 0.006 * torch.rand(tiles, k // case["group"], 16, generator=g, device="cuda")).half()
        s["x"] = _normal(g, case["rows"], k)
        s["norm"] = 1.0 + _normal(g, k, std=0.1) if case["norm"] else None
        s["y"] = torch.zeros(case["rows"], n // 2 if swiglu else n, device="cuda")
    return s


def work(case):
    kind = case["kind"]
    eb = 2 if case.get("cache") == "f16" else 4
    if kind in ("attn", "append"):
        past, new = _pasts(case), _news(case)
        rows = sum(new)
        if kind == "append":
            return {"bytes": rows * (4 * (Q_DIM + 2 * KV_DIM) + 4 * Q_DIM + 2 * KV_DIM * eb), "flops": 8 * rows * Q_DIM}
        pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
        keys = sum(p + n for p, n in zip(past, new))
        return {"bytes": keys * 2 * KV_DIM * eb + 8 * rows * Q_DIM, "flops": 4 * Q_DIM * pairs}
    page = case.get("page", 0) * 2 * KV_DIM * eb * case.get("layers", 0)
    if kind == "fork":
        ps, n, prefix = case["page"], case["beams"], case["prefix"]
        copies = n if prefix % ps else 0
        return {"bytes": 2 * copies * page + 4 * n * 3 * (prefix // ps + 2), "flops": 0}
    if kind == "compact":
        counts = [-(-max(1, case["longest"] - (37 * i) % case["longest"]) // case["page"]) for i in range(case["seqs"])]
        live = sum(counts)
        pages = max(live + 1, live * 100 // (100 - case["free"]))
        return {"bytes": 2 * page * live * (pages - live) // pages + 8 * (pages + live), "flops": 0}
    n, k, swiglu = MATRICES[case["matrix"]]
    out = n // 2 if swiglu else n
    return {"bytes": n * k // 2 + 2 * n * k // case["group"] + 4 * case["rows"] * (k + out),
            "flops": 2 * n * k * case["rows"]}


# ------------------------------------------------------------------------------------------ plain forms
def _row_places(s):
    """The sequence and the position of every row."""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["row_start"][1:].long(), row, right=True)
    return seq, s["n_past"].long()[seq] + row - s["row_start"].long()[seq]


def _plain_attn(s):
    case = s["case"]
    n, ps = case["seqs"], case["page"]
    k, v = s["pages"][s["layer"]]
    table = s["tables"].long().clamp(min=0)
    k, v = (x[table].permute(0, 2, 1, 3, 4).reshape(n, KV_HEADS, -1, DIM).float() for x in (k, v))
    t = torch.arange(s["max_new"], device="cuda")
    start = s["row_start"].long()
    row = (start[:-1, None] + t).clamp(max=s["rows"] - 1)
    q = s["q"][row].view(n, -1, KV_HEADS, GROUP, DIM).permute(0, 2, 1, 3, 4).reshape(n, KV_HEADS, -1, DIM)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * SCALE
    seen = torch.arange(k.shape[2], device="cuda") <= (s["n_past"].long()[:, None] + t)[..., None]
    hidden = ~seen[:, None, :, None, :]
    scores = scores.view(n, KV_HEADS, -1, GROUP, k.shape[2]).masked_fill_(hidden, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = torch.matmul(e.view(n, KV_HEADS, -1, k.shape[2]), v) / e.sum(-1).view(n, KV_HEADS, -1, 1)
    o = o.view(n, KV_HEADS, -1, GROUP, DIM).permute(0, 2, 1, 3, 4).reshape(n, -1, Q_DIM)
    seq, pos = _row_places(s)
    s["out"].copy_(o[seq, pos - s["n_past"].long()[seq]])
    return s["out"]


def _plain_append(s):
    seq, pos = _row_places(s)
    rows, ps = s["rows"], s["case"]["page"]
    q, k, v = (x.view(rows, -1, DIM) for x in s["qkv"].split([Q_DIM, KV_DIM, KV_DIM], 1))
    freq = torch.exp(-math.log(THETA) * torch.arange(0, DIM, 2, device="cuda", dtype=torch.float64) / DIM)
    angle = pos[:, None].double() * freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def rotated(x, w):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    s["q"].copy_(rotated(q, s["q_norm"]).view(rows, Q_DIM))
    page = s["tables"].long()[seq, pos // ps]
    pool = s["pages"][s["layer"]]
    pool[0][page, :, pos % ps] = rotated(k, s["k_norm"]).to(pool.dtype)
    pool[1][page, :, pos % ps] = v.to(pool.dtype)
    return {"q": s["q"], "pages": s["pages"]}


def _plain_fork(s):
    ps, refs, tables, beams = s["case"]["page"], s["refs"], s["tables"], s["beams"].long()
    # free: every entry of the beams' rows gives its page back
    old = tables[beams]
    refs.index_add_(0, old.clamp(min=0).flatten().long(), -(old >= 0).int().flatten())
    # fork: the parent's entries up to the last page that holds a position
    col = torch.arange(tables.shape[1], device="cuda")
    held = col < ((s["lens"] + ps - 1) // ps)[:, None]
    new = torch.where(held, tables[s["parents"].long()], -1)
    refs.index_add_(0, new.clamp(min=0).flatten().long(), (new >= 0).int().flatten())
    # extend: a written page that others hold too is copied, pages that are not there are taken; lowest free first
    first, last = s["lens"] // ps, (s["lens"] + s["ones"] + ps - 1) // ps
    written = new.gather(1, first[:, None].long())[:, 0]
    same = (written[:, None] == written[None, :]).tril(-1) & (written >= 0)
    copied = (written >= 0) & (refs[written.clamp(min=0).long()] - same.sum(1) > 1)
    wanted = ((col >= first[:, None]) & (col < last[:, None]) & (new < 0)) | (copied[:, None] & (col == first[:, None]))
    free = refs <= 0
    lowest = torch.argsort((~free).int(), stable=True).int()
    rank = wanted.flatten().cumsum(0).view_as(wanted) - 1
    given = torch.where(wanted, lowest[rank.clamp(min=0)], new)
    taken = given.gather(1, first[:, None].long())[:, 0]
    refs.index_add_(0, written.clamp(min=0).long(), -copied.int())
    refs.index_add_(0, given.clamp(min=0).flatten().long(), wanted.int().flatten())
    tables[beams] = given
    to, source = taken[copied].long(), written[copied].long()
    s["pages"][:, :, to] = s["pages"][:, :, source]
    s["missing"].copy_((wanted.sum() - free.sum()).clamp(min=0))
    return {"pages": s["pages"], "tables": tables, "refs": refs, "missing": s["missing"]}


def _plain_compact(s):
    refs, tables = s["refs"], s["tables"]
    ids = torch.arange(refs.numel(), device="cuda")
    used = refs > 0
    live = used.sum()
    holes, movers = ids[~used & (ids < live)], ids[used & (ids >= live)]
    place = ids.clone()
    place[movers] = holes
    s["pages"][:, :, holes] = s["pages"][:, :, movers]
    s["refs_out"].copy_(refs)
    s["refs_out"][holes] = refs[movers]
    s["refs_out"][movers] = 0
    s["tables_out"].copy_(torch.where(tables >= 0, place[tables.clamp(min=0).long()], -1))
    s["live"].copy_(live)
    return {"pages": s["pages"], "tables": s["tables_out"], "refs": s["refs_out"], "live": s["live"]}


def _weights(s, dtype):
    """W [rows][columns] of its packed form: lane 16 j + r of a 1 KB block holds row r, columns 32 w + 8 j + e of the
    block in its word w, column e in bits 4 (e / 2) + 16 (e % 2)."""
    n, k, _ = MATRICES[s["case"]["matrix"]]
    group = s["case"]["group"]
    shift = torch.tensor([4 * (e // 2) + 16 * (e % 2) for e in range(8)], device="cuda", dtype=torch.int32)
    words = s["weights"].view(torch.int32).view(n // 16, k // 128, 4, 16, 4, 1)
    q = ((words >> shift) & 15).to(dtype) - 8
    q = q.permute(0, 3, 1, 4, 2, 5).reshape(n // 16, 16, k // group, group)
    d = s["scales"].to(dtype).transpose(1, 2)
    return (q * d[..., None]).view(n, k)


def _plain_q4(s):
    x = s["x"]
    if s["norm"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["norm"]
    y = torch.matmul(x, _weights(s, torch.float32).t())
    if MATRICES[s["case"]["matrix"]][2]:
        gate, up = y.chunk(2, 1)
        y = gate / (1 + torch.exp(-gate)) * up
    s["y"].copy_(y)
    return s["y"]


# ------------------------------------------------------------------------------------------ the framework's calls
def _calls(s):
    """The entry points' arguments, which a program keeps for as long as it keeps its buffers."""
    import ctypes as C

    if os.path.join(os.getcwd(), "qwenasr.cpp_amd") not in sys.path:
        sys.path.insert(0, os.path.join(os.getcwd(), "qwenasr.cpp_amd"))
    import qwenasr_amd as qa

    case, lib = s["case"], qa.lib

    def p(t):
        return C.c_void_p(t.data_ptr() if t is not None else None)

    def space(n):
        s["workspace"] = torch.empty(max(int(n), 256), dtype=torch.uint8, device="cuda")
        return p(s["workspace"]), s["workspace"].numel()

    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    if case["kind"] == "q4":
        n, k, swiglu = MATRICES[case["matrix"]]
        return [(lib.qa_gemv_q4, (p(s["weights"]), p(s["scales"]), case["group"], n // 2 if swiglu else n, k, p(s["x"]),
                                  case["rows"], p(s["y"]), 2 if swiglu else 0, p(s["norm"]), EPS, stream))], s["y"]
    pool = s["pages"]
    kv_type = qa.QA_CACHE_F16 if case["cache"] == "f16" else qa.QA_CACHE_F32
    layout = qa.KvLayout(pool.shape[0], pool.shape[2], KV_HEADS, DIM, case["page"], kv_type)
    lay = C.byref(layout)
    rows, stride = s["tables"].shape
    s["keep"] = [layout]
    if case["kind"] in ("attn", "append"):
        batch = qa.PagedBatch(p(s["tables"]), p(s["n_past"]), p(s["row_start"]), rows, stride, s["rows"], s["max_new"],
                              s["max_len"])
        s["keep"].append(batch)
        b = C.byref(batch)
        if case["kind"] == "attn":
            ws = space(lib.qa_paged_attn_workspace_bytes(lay, b, HEADS))
            return [(lib.qa_paged_attn, (p(s["q"]), p(pool), lay, s["layer"], b, HEADS, SCALE, p(s["out"]), *ws,
                                         stream))], s["out"]
        return [(lib.qa_paged_append, (p(s["qkv"]), p(s["q_norm"]), p(s["k_norm"]), p(s["q"]), p(pool), lay, s["layer"],
                                       b, HEADS, THETA, EPS, stream))], {"q": s["q"], "pages": pool}
    if case["kind"] == "fork":
        n = case["beams"]
        table = (p(s["refs"]), pool.shape[2], p(s["tables"]), rows, stride)
        ws = space(lib.qa_pages_workspace_bytes(lay))
        return [
            (lib.qa_pages_free, (*table, case["page"], p(s["beams"]), None, n, stream)),
            (lib.qa_pages_fork, (*table, case["page"], p(s["parents"]), p(s["beams"]), p(s["lens"]), n, stream)),
            (lib.qa_pages_extend, (p(pool), lay, p(s["refs"]), p(s["tables"]), rows, stride, p(s["beams"]), p(s["lens"]),
                                   p(s["ones"]), n, p(s["missing"]), *ws, stream)),
        ], {"pages": pool, "tables": s["tables"], "refs": s["refs"], "missing": s["missing"]}
    ws = space(lib.qa_pages_workspace_bytes(lay))
    return [(lib.qa_pages_compact, (p(pool), lay, p(s["refs"]), p(s["tables"]), rows, stride, p(s["refs_out"]),
                                    p(s["tables_out"]), p(s["live"]), *ws, stream))], {
        "pages": pool, "tables": s["tables_out"], "refs": s["refs_out"], "live": s["live"]}


def _own(s):
    if "calls" not in s:
        s["calls"], s["result"] = _calls(s)
    for call, arguments in s["calls"]:
        if call(*arguments) != 0:
            import qwenasr_amd as qa

            raise RuntimeError(qa.lib.qa_last_error().decode())
    return s["result"]


_PLAIN = {"attn": _plain_attn, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact, "q4": _plain_q4}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(s)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "q4":
        return _exact_q4(s)
    return None  # pages are moved, tables and counts are whole numbers: nothing is computed


def _lists(s):
    return s["tables"].tolist(), s["n_past"].tolist(), s["row_start"].tolist()


def _exact_attn(s):
    tables, past, start = _lists(s)
    ps = s["case"]["page"]
    out = torch.zeros(s["rows"], HEADS, DIM, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(-1, HEADS, DIM)
    for i, (n_past, row) in enumerate(zip(past, tables)):
        n = start[i + 1] - start[i]
        length = n_past + n
        ids = row[:-(-length // ps)]
        late = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(n_past + 1)
        for h in range(HEADS):
            k, v = (s["pages"][s["layer"], kv, ids, h // GROUP].reshape(-1, DIM)[:length].double() for kv in (0, 1))
            scores = (q[start[i]:start[i + 1], h] @ k.t() / math.sqrt(DIM)).masked_fill(late, -math.inf)
            out[start[i]:start[i + 1], h] = torch.softmax(scores, -1) @ v
    return out.view(-1, Q_DIM)


def _exact_append(s):
    tables, past, start = _lists(s)
    ps = s["case"]["page"]
    x = s["qkv"].double().view(s["rows"], -1, DIM)
    at = torch.cat([torch.arange(start[i + 1] - start[i], device="cuda") + past[i] for i in range(len(past))])
    turn = at.double()[:, None, None] * THETA ** (-torch.arange(0, DIM, 2, device="cuda", dtype=torch.float64) / DIM)
    turn = torch.polar(torch.ones_like(turn), turn)

    def rotated(y, w):
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
        z = torch.complex(y[..., :DIM // 2], y[..., DIM // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    q, k, v = rotated(x[:, :HEADS], s["q_norm"]), rotated(x[:, HEADS:HEADS + KV_HEADS], s["k_norm"]), x[:, HEADS + KV_HEADS:]
    pages = s["pages"].double()
    for i, row in enumerate(tables):
        for j in range(past[i] // ps, -(-(past[i] + start[i + 1] - start[i]) // ps)):
            lo, hi = max(j * ps, past[i]), min((j + 1) * ps, past[i] + start[i + 1] - start[i])
            a = start[i] + lo - past[i]
            for kv, y in ((0, k), (1, v)):
                pages[s["layer"], kv, row[j], :, lo - j * ps:hi - j * ps] = y[a:a + hi - lo].transpose(0, 1)
    return {"q": q.reshape(-1, Q_DIM), "pages": pages}


def _exact_q4(s):
    n, k, swiglu = MATRICES[s["case"]["matrix"]]
    x = s["x"].double()
    if s["norm"] is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * s["norm"].double()
    y = torch.zeros(s["case"]["rows"], n, dtype=torch.float64, device="cuda")
    low = s["weights"].view(n // 16, k // 128, 4, 16, 4, 4).to(torch.int16)  # block, column block, j, row, word, byte
    per = s["case"]["group"]
    for j in range(4):
        for word in range(4):
            for e in range(8):
                bit = 4 * (e // 2) + 16 * (e % 2)
                q = ((low[:, :, j, :, word, bit // 8] >> (bit % 8)) & 15).double() - 8
                cols = torch.arange(k // 128, device="cuda") * 128 + 32 * word + 8 * j + e
                d = s["scales"].double()[:, torch.div(cols, per, rounding_mode="floor")]
                y += x[:, cols] @ (q * d).transpose(1, 2).reshape(n, -1).t()
    if swiglu:
        gate, up = y[:, :n // 2], y[:, n // 2:]
        y = gate * torch.sigmoid(gate) * up
    return y
