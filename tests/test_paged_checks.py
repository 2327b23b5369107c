"""What the paged-cache and 4-bit entry points refuse, and the bounds that turn device data into addresses, on the CPU."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import paged_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20   # an aligned address that no refused call reads


def refused(qa, rc, text):
    assert rc == qa.QA_ERR_INVALID
    assert text in qa.lib.qa_last_error().decode(), qa.lib.qa_last_error().decode()


def batch(qa, **kw):
    d = dict(tables=P, n_past=P, row_start=P, n_seqs=2, table_stride=4, n_rows=2, max_tokens=1, max_len=64)
    d.update(kw)
    return qa.PagedBatch(*(d[n] for n, _ in qa.PagedBatch._fields_))


def attn(qa, lay, b, q=P, pages=P, layer=0, heads=16, scale=1.0, out=P, ws=None, ws_bytes=0):
    return qa.lib.qa_paged_attn(q, pages, C.byref(lay) if lay else None, layer, C.byref(b) if b else None, heads, scale, out, ws,
                                ws_bytes, None)


def append(qa, lay, b, qkv=P, qn=P, kn=P, q=P, pages=P, layer=0, heads=16, theta=1e6):
    return qa.lib.qa_paged_append(qkv, qn, kn, q, pages, C.byref(lay), layer, C.byref(b), heads, theta, 1e-6, None)


def test_attention_and_append_refusals(qa):
    good = ref.layout(qa, 2, 8, 8, 16, True)
    for call in (attn, append):
        for page in (1, 8, 24, 512):
            refused(qa, call(qa, ref.layout(qa, 2, 8, 8, page, True), batch(qa)), "positions")
        refused(qa, call(qa, qa.KvLayout(2, 8, 8, 64, 16, qa.QA_CACHE_F16), batch(qa)), "head_dim")
        refused(qa, call(qa, qa.KvLayout(2, 0, 8, 128, 16, qa.QA_CACHE_F16), batch(qa)), "KV-cache configuration")
        refused(qa, call(qa, good, batch(qa), layer=2), "layer")
        refused(qa, call(qa, good, batch(qa), layer=-1), "layer")
        for heads in (0, -16, 12, 8 * 17):
            refused(qa, call(qa, good, batch(qa), heads=heads), "heads")
        for kw in (dict(n_seqs=0), dict(n_seqs=-1), dict(table_stride=0), dict(table_stride=(1 << 26) + 1)):
            refused(qa, call(qa, good, batch(qa, **kw)), "page table")
        for kw in (dict(n_rows=-1), dict(n_rows=1 << 30), dict(max_tokens=-1), dict(max_len=-1)):
            refused(qa, call(qa, good, batch(qa, **kw)), "out of range")
        for kw in (dict(tables=None), dict(n_past=None), dict(row_start=None)):
            refused(qa, call(qa, good, batch(qa, **kw)), "null pointer")
        assert call(qa, good, batch(qa, n_rows=0, tables=None, n_past=None, row_start=None)) == qa.QA_OK   # nothing to do
    refused(qa, attn(qa, None, batch(qa)), "null KV layout")
    refused(qa, attn(qa, good, None), "null batch")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(qa, attn(qa, good, batch(qa), scale=scale), "scale")
    for kw in (dict(q=None), dict(pages=None), dict(out=None), dict(ws_bytes=64)):
        refused(qa, attn(qa, good, batch(qa), **kw), "null pointer")
    for kw in (dict(q=P + 4), dict(pages=P + 8), dict(out=P + 4), dict(ws=P + 4, ws_bytes=64)):
        refused(qa, attn(qa, good, batch(qa), **kw), "aligned")
    refused(qa, attn(qa, good, batch(qa, n_rows=(1 << 30) - 1)), "too many rows")
    for kw in (dict(qkv=None), dict(qn=None), dict(kn=None), dict(q=None), dict(pages=None)):
        refused(qa, append(qa, good, batch(qa), **kw), "null pointer")
    for theta in (0.0, -1.0, float("nan")):
        refused(qa, append(qa, good, batch(qa), theta=theta), "rope_theta")


def test_attention_workspace(qa):
    lay = ref.layout(qa, 2, 1024, 8, 16, True)

    def need(**kw):
        return qa.lib.qa_paged_attn_workspace_bytes(C.byref(lay), C.byref(batch(qa, **kw)), 16)

    assert need(n_rows=0) == 0
    assert need(n_seqs=1, n_rows=1, max_len=16) == 0                                # one key range
    one = need(n_seqs=1, n_rows=1, table_stride=300, max_len=4000)
    assert one > 0 and one % (16 * 130 * 4) == 0 and one <= 64 * 16 * 130 * 4       # at most 64 ranges of 16 heads
    assert need(n_seqs=1, n_rows=1, table_stride=300, max_len=0) == need(n_seqs=1, n_rows=1, table_stride=300, max_len=4800)
    assert need(n_seqs=0) == 0 and qa.lib.qa_paged_attn_workspace_bytes(None, None, 16) == 0


def test_page_bookkeeping_refusals(qa):
    lib = qa.lib
    lay = ref.layout(qa, 2, 8, 8, 16, True)
    ws = lib.qa_pages_workspace_bytes(C.byref(lay))
    assert ws >= 3 * 8 * 4
    assert lib.qa_pages_workspace_bytes(C.byref(ref.layout(qa, 2, 8, 8, 17, True))) == 0

    def extend(lay=lay, pages=P, refs=P, tables=P, n_rows=2, stride=4, rows=P, past=P, new=P, n=2, missing=P, w=P, wb=ws):
        return lib.qa_pages_extend(pages, C.byref(lay), refs, tables, n_rows, stride, rows, past, new, n, missing, w, wb, None)

    def fork(refs=P, n_pages=8, tables=P, n_rows=2, stride=4, page=16, src=P, dst=P, length=P, n=1):
        return lib.qa_pages_fork(refs, n_pages, tables, n_rows, stride, page, src, dst, length, n, None)

    def release(refs=P, n_pages=8, tables=P, n_rows=2, stride=4, page=16, rows=P, n=1):
        return lib.qa_pages_free(refs, n_pages, tables, n_rows, stride, page, rows, None, n, None)

    def copy(lay=lay, pages=P, src=P, dst=P, n=1):
        return lib.qa_pages_copy(pages, C.byref(lay), src, dst, n, None)

    def compact(lay=lay, pages=P, refs=P, tables=P, n_rows=2, stride=4, ro=P, to=P, live=P, w=P, wb=ws):
        return lib.qa_pages_compact(pages, C.byref(lay), refs, tables, n_rows, stride, ro, to, live, w, wb, None)

    bad = ref.layout(qa, 2, 8, 8, 20, True)
    for call in (extend, copy, compact):
        refused(qa, call(lay=bad), "positions")
        refused(qa, call(pages=None), "null pointer")
        refused(qa, call(pages=P + 4), "aligned")
        refused(qa, call(lay=ref.layout(qa, 40000, 8, 8, 16, True)), "layers")
    for call in (fork, release):
        refused(qa, call(page=20), "positions")
        refused(qa, call(n_pages=0), "positions")
    for call in (extend, fork, release, compact):
        for kw in (dict(n_rows=0), dict(stride=0), dict(stride=1 << 27)):
            refused(qa, call(**kw), "page table")
        for kw in (dict(refs=None), dict(tables=None)):
            refused(qa, call(**kw), "null pointer")
    for call in (extend, fork, release, copy):
        for n in (-1, 1025):
            refused(qa, call(n=n), "1024")
    for kw in (dict(past=None), dict(new=None), dict(missing=None)):
        refused(qa, extend(**kw), "null pointer")
    for kw in (dict(src=None), dict(dst=None), dict(length=None)):
        refused(qa, fork(**kw), "null pointer")
    refused(qa, release(rows=None), "null pointer")
    for kw in (dict(src=None), dict(dst=None)):
        refused(qa, copy(**kw), "null pointer")
    for kw in (dict(ro=None), dict(to=None), dict(live=None)):
        refused(qa, compact(**kw), "null pointer")
    for call in (extend, compact):
        refused(qa, call(w=None), "workspace")
        refused(qa, call(wb=ws - 1), "workspace")
    assert fork(n=0) == release(n=0) == copy(n=0) == qa.QA_OK


def test_q4_refusals_and_sizes(qa):
    lib = qa.lib
    assert lib.qa_q4_weight_bytes(151936, 2048) == 151936 * 1024
    assert lib.qa_q4_weight_bytes(17, 128) == 32 * 64 and lib.qa_q4_scale_count(17, 256, 64) == 32 * 4
    assert lib.qa_q4_weight_bytes(16, 100) == 0 and lib.qa_q4_scale_count(16, 128, 16) == 0

    def gemv(w=P, s=P, group=32, out=32, k=256, x=P, rows=1, y=P, epi=0, norm=None):
        return lib.qa_gemv_q4(w, s, group, out, k, x, rows, y, epi, norm, 1e-6, None)

    def pack(src=P, out=32, k=256, group=32, w=P, s=P):
        return lib.qa_pack_q4(src, out, k, group, w, s, None)

    for call in (gemv, pack):
        for kw in (dict(out=0), dict(out=-1), dict(k=0), dict(k=64), dict(k=200), dict(out=(1 << 24) + 1), dict(k=(1 << 20) + 128)):
            refused(qa, call(**kw), "in_dim")
        for group in (0, 16, 48, 256):
            refused(qa, call(group=group), "groups")
        for kw in (dict(w=None), dict(s=None)):
            refused(qa, call(**kw), "null pointer")
        for kw in (dict(w=P + 8), dict(s=P + 4)):
            refused(qa, call(**kw), "aligned")
    for rows in (0, -1, 33):
        refused(qa, gemv(rows=rows), "rows")
    for epi in (-1, 3):
        refused(qa, gemv(epi=epi), "epilogue")
    refused(qa, gemv(out=40, epi=2), "SwiGLU")
    for kw in (dict(x=None), dict(y=None)):
        refused(qa, gemv(**kw), "null pointer")
    for kw in (dict(x=P + 4), dict(norm=P + 4)):
        refused(qa, gemv(**kw), "aligned")
    refused(qa, pack(src=None), "null pointer")


BOUNDS = r"""
#include "paged.hpp"
#include <cstdio>
#include <vector>
using namespace qa;
int main() {
    const int32_t table[4] = {3, -1, 8, 7};
    for (int pos : {-2147483647, -1, 0, 15, 16, 31, 32, 48, 63, 64, 2147483647}) std::printf("%d ", page_of(table, 4, 4, 8, pos));
    std::printf("\n");
    for (int v : {-2147483647, -5, 0, 7, 1 << 30, 2147483647}) std::printf("%d ", bounded_past(v));
    std::printf("\n");
    const int r[][3] = {{0, 5, 9}, {5, 12, 9}, {9, 12, 9}, {4, 4, 9}, {6, 2, 9}, {-3, 4, 9}, {0, 2147483647, 9}, {2147483647, 2147483647, 9}};
    for (auto & a : r) std::printf("%d ", rows_between(a[0], a[1], a[2]));
    std::printf("\n");
    for (int p : {16, 32, 64, 128, 256}) std::printf("%d ", page_shift_of(p));
    std::printf("\n");
    return 0;
}
"""


def test_device_data_is_bounded(tmp_path):
    """Page numbers, positions, lengths and row starts of any value, through the functions that the kernels use."""
    src = tmp_path / "bounds.cpp"
    src.write_text(BOUNDS)
    exe = tmp_path / "bounds"
    pkg = os.path.join(ROOT, "qwenasr.cpp_amd")
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{ROOT}/include", f"-I{pkg}/csrc", str(src),
                    "-o", str(exe), f"-L{pkg}", "-lqwenasr_amd", "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{pkg}:/opt/rocm/lib",
                    "-Wl,--unresolved-symbols=ignore-all"], check=True, capture_output=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    got = [[int(v) for v in line.split()] for line in lines]
    assert got[0] == [-1, -1, 3, 3, -1, -1, -1, 7, 7, -1, -1]     # page 8 of 8 is no page
    assert got[1] == [-(1 << 30), -5, 0, 7, 1 << 30, 1 << 30]
    assert got[2] == [5, 4, 0, 0, 0, 0, 9, 0]
    assert got[3] == [4, 5, 6, 7, 8]


def test_plain_bookkeeping_by_hand():
    """The plain statements that the GPU tests compare with, on cases small enough to read."""
    refs = np.array([2, 0, 2, 0, 0], np.int32)
    tables = np.array([[0, 2, -1], [0, 2, -1]], np.int32)
    r, t, copies, missing = ref.extend(refs, tables, 16, [0, 1], [20, 20], [1, 1])
    assert missing == 0 and copies == [(2, 1)] and t.tolist() == [[0, 1, -1], [0, 2, -1]] and r.tolist() == [2, 1, 1, 0, 0]
    r, t, copies, missing = ref.extend(refs, tables, 16, [0, 1], [20, 32], [60, 16])
    assert missing == 0 and copies == [(2, 1)] and t.tolist() == [[0, 1, 3], [0, 2, 4]] and r.tolist() == [2, 1, 1, 1, 1]
    r, t, copies, missing = ref.extend(refs, np.hstack([tables, tables[:, 2:]]), 16, [0, 1], [20, 20], [44, 44])
    assert missing == 2 and copies == [] and r.tolist() == refs.tolist()
    r, t = ref.free(refs, tables, 16, [1], [16])
    assert r.tolist() == [2, 0, 1, 0, 0] and t.tolist() == [[0, 2, -1], [0, -1, -1]]
    r, t = ref.fork(refs, tables, 16, [0], [1], [16])
    assert r.tolist() == [2, 0, 1, 0, 0] and t.tolist() == [[0, 2, -1], [0, -1, -1]]
    r, t, moves, live = ref.compact(np.array([0, 1, 0, 2, 1], np.int32), np.array([[1, 3], [4, 3]], np.int32))
    assert live == 3 and moves == [(3, 0), (4, 2)] and t.tolist() == [[1, 0], [2, 0]] and r.tolist() == [2, 1, 1, 0, 0]
