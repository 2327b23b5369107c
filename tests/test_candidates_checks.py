"""What the entry points of the 8-bit cache, of drafted trees and of beam selection refuse, on the CPU."""
import ctypes as C

import pytest

import paged_ref as ref
from test_paged_checks import P, append, attn, batch, refused


def q8(qa, layers=2, pages=8, heads=8, dim=128, page=16):
    return qa.KvLayout(layers, pages, heads, dim, page, qa.QA_CACHE_Q8)


def test_layout(qa):
    lib = qa.lib
    lay = q8(qa, 28, 10, 8, 128, 64)
    assert lib.qa_kv_layout_check(C.byref(lay)) == qa.QA_OK and lib.qa_kv_elem_bytes(qa.QA_CACHE_Q8) == 1
    block = 8 * 64 * 132
    assert lib.qa_kv_cache_bytes(C.byref(lay)) == 28 * 2 * 10 * block
    assert lib.qa_kv_slot_index(C.byref(lay), 3, 1, 7, 5, 60, 9) == ((3 * 2 + 1) * 10 + 7) * block + (5 * 64 + 60) * 128 + 9
    for bad in (q8(qa, dim=64), q8(qa, page=17), q8(qa, page=8), q8(qa, page=512), q8(qa, page=4169)):
        assert lib.qa_kv_cache_bytes(C.byref(bad)) == 0
        refused(qa, lib.qa_kv_layout_check(C.byref(bad)), "8 bits")
    for bad in (qa.KvLayout(2, 8, 8, 128, 16, 3), qa.KvLayout(2, 8, 8, 128, 16, -1), q8(qa, pages=0)):
        refused(qa, lib.qa_kv_layout_check(C.byref(bad)), "KV-cache configuration")
        assert lib.qa_kv_cache_bytes(C.byref(bad)) == 0
    refused(qa, attn(qa, q8(qa, page=24), batch(qa)), "8 bits")
    refused(qa, append(qa, q8(qa, dim=64), batch(qa)), "8 bits")


def test_the_flat_cache_has_no_8_bits(qa):
    lay = C.byref(q8(qa, page=256))
    lib = qa.lib
    refused(qa, lib.qa_kv_append(P, P, P, P, P, lay, 0, P, 1, 1, 16, 1e6, 1e-6, None), "8 bits")
    refused(qa, lib.qa_decode_attn(P, P, lay, 0, P, 1, 10, 16, 0.1, P, P, 1 << 30, None), "8 bits")
    refused(qa, lib.qa_decode_step_attn(P, P, P, P, lay, 0, P, 1, 10, 16, 1e6, 1e-6, 0.1, P, P, 1 << 30, None), "8 bits")
    refused(qa, lib.qa_decode_step_attn_noalloc(P, P, P, P, lay, 0, P, 1, 10, 16, 1e6, 1e-6, 0.1, P, None), "8 bits")
    refused(qa, lib.qa_prefill_attn(P, P, lay, 0, 0, 0, 4, 16, 0.1, P, P, 1 << 30, None), "8 bits")


def test_read(qa):
    def read(lay=q8(qa), b=batch(qa), pages=P, layer=0, k=P, v=P, kind=qa.QA_CACHE_F16):
        return qa.lib.qa_paged_read(pages, C.byref(lay) if lay else None, layer, C.byref(b) if b else None, k, v, kind, None)

    refused(qa, read(lay=None), "null KV layout")
    refused(qa, read(b=None), "null batch")
    refused(qa, read(layer=2), "layer")
    for kind in (qa.QA_CACHE_Q8, 3, -1):
        refused(qa, read(kind=kind), "f32 or f16")
    refused(qa, read(pages=None), "null pointer")
    refused(qa, read(b=batch(qa, row_start=None)), "null pointer")
    for kw in (dict(pages=P + 8), dict(k=P + 4), dict(v=P + 8)):
        refused(qa, read(**kw), "aligned")
    assert read(k=None, v=None) == qa.QA_OK and read(b=batch(qa, n_rows=0)) == qa.QA_OK       # nothing to do


def test_trees(qa):
    lib = qa.lib
    lay = ref.layout(qa, 2, 8, 8, 16, True)

    def tree_attn(b=batch(qa), mask=P, words=1, q=P, heads=16, layout=lay, out=P, scale=1.0):
        return lib.qa_paged_tree_attn(q, P, C.byref(layout), 0, C.byref(b) if b else None, mask, words, heads, scale, out, None, 0, None)

    def prepare(b=batch(qa), parents=P, mask=P, words=1, depth=P):
        return lib.qa_tree_prepare(C.byref(b) if b else None, parents, mask, words, depth, None)

    def accept(b=batch(qa), parents=P, ids=P, picks=P, path=P, kept=P, nxt=P):
        return lib.qa_tree_accept(C.byref(b) if b else None, parents, ids, picks, path, kept, nxt, None)

    def keep(b=batch(qa), layout=lay, pages=P, path=P, kept=P):
        return lib.qa_paged_keep(pages, C.byref(layout) if layout else None, C.byref(b) if b else None, path, kept, None)

    for call in (tree_attn, prepare):
        for words in (0, -1, 33):
            refused(qa, call(words=words), "words")
        refused(qa, call(mask=None), "null pointer")
    for call in (tree_attn, prepare, accept, keep):
        refused(qa, call(b=None), "null batch")
        refused(qa, call(b=batch(qa, n_rows=(1 << 24) + 1)), "out of range")
        refused(qa, call(b=batch(qa, n_rows=-1)), "out of range")
        refused(qa, call(b=batch(qa, row_start=None)), "null pointer")
    for call in (tree_attn, prepare, keep):
        assert call(b=batch(qa, n_rows=0, row_start=None, tables=None, n_past=None)) == qa.QA_OK
    refused(qa, tree_attn(heads=12), "heads")
    refused(qa, tree_attn(scale=0.0), "scale")
    refused(qa, tree_attn(q=P + 4), "aligned")
    refused(qa, tree_attn(out=None), "null pointer")
    for kw in (dict(parents=None), dict(depth=None)):
        refused(qa, prepare(**kw), "null pointer")
    for kw in (dict(parents=None), dict(ids=None), dict(picks=None), dict(path=None), dict(kept=None), dict(nxt=None)):
        refused(qa, accept(**kw), "null pointer")
    refused(qa, accept(b=batch(qa, n_seqs=0)), "out of range")
    refused(qa, keep(b=batch(qa, n_seqs=65536)), "sequences")
    refused(qa, keep(layout=None), "null KV layout")
    refused(qa, keep(pages=P + 8), "aligned")
    for kw in (dict(pages=None), dict(path=None), dict(kept=None)):
        refused(qa, keep(**kw), "null pointer")
    b = batch(qa)
    refused(qa, lib.qa_paged_tree_append(P, P, P, P, P, C.byref(lay), 0, C.byref(b), None, 16, 1e6, 1e-6, None), "null pointer")
    refused(qa, lib.qa_paged_tree_append(P, P, P, P, P, C.byref(lay), 5, C.byref(b), P, 16, 1e6, 1e-6, None), "layer")
    refused(qa, lib.qa_paged_tree_append(P, P, P, P, P, C.byref(lay), 0, None, P, 16, 1e6, 1e-6, None), "null batch")


def test_beams(qa):
    lib = qa.lib
    need = lib.qa_beam_select_workspace_bytes(2, 4, 1000)

    def select(logits=P, groups=2, width=4, vocab=1000, scores=P, done=None, stops=P, n_stop=2, p=P, t=P, s=P, d=P, ws=P, size=need):
        return lib.qa_beam_select(logits, groups, width, vocab, scores, done, stops, n_stop, p, t, s, d, ws, size, None)

    def reorder(refs=P, n_pages=8, tables=P, n_rows=4, stride=4, page=16, rows=P, parents=P, lens=P, n=2, ids=P, ids_stride=9, tokens=P, at=P):
        return lib.qa_beam_reorder(refs, n_pages, tables, n_rows, stride, page, rows, parents, lens, n, ids, ids_stride, tokens, at, None)

    assert need > 0 and lib.qa_beam_select_workspace_bytes(2, 0, 1000) == 0 and lib.qa_beam_select_workspace_bytes(2, 4, 3) == 0
    for width in (0, -1, 65):
        refused(qa, select(width=width), "beams")
    for groups in (-1, 16384):
        refused(qa, select(groups=groups), "rows")
    for vocab in (3, 0, -5, (1 << 30) + 1):
        refused(qa, select(vocab=vocab), "vocabulary")
    for n in (-1, 65):
        refused(qa, select(n_stop=n), "stop ids")
    for kw in (dict(logits=None), dict(scores=None), dict(stops=None), dict(p=None), dict(t=None), dict(s=None), dict(d=None)):
        refused(qa, select(**kw), "null pointer")
    for kw in (dict(ws=None), dict(size=need - 1), dict(size=0)):
        refused(qa, select(**kw), "workspace")
    refused(qa, select(ws=P + 8), "aligned")
    assert select(groups=0) == qa.QA_OK
    for n in (-1, 1025):
        refused(qa, reorder(n=n), "1024")
    for kw in (dict(refs=None), dict(tables=None), dict(parents=None), dict(lens=None), dict(at=None)):
        refused(qa, reorder(**kw), "null pointer")
    for page in (0, 8, 24, 512):
        refused(qa, reorder(page=page), "positions")
    refused(qa, reorder(n_pages=0), "positions")
    refused(qa, reorder(n_rows=0), "no rows")
    for kw in (dict(stride=0), dict(stride=(1 << 26) + 1)):
        refused(qa, reorder(**kw), "page table")
    for stride in (0, -1, (1 << 30) + 1):
        refused(qa, reorder(ids_stride=stride), "ids_stride")
    assert reorder(n=0) == qa.QA_OK and reorder(refs=None, tables=None, ids=None) == qa.QA_OK
