// Device side of a ragged batch: which sequence a row belongs to.
#pragma once

#include "paged.hpp"

namespace qa {

struct PagedSeqs {
    const int32_t * tables;
    const int32_t * n_past;
    const int32_t * row_start;
    int32_t n_seqs, table_stride, n_rows;
};

inline PagedSeqs paged_seqs(const qa_paged_batch & b) {
    return PagedSeqs{b.tables, b.n_past, b.row_start, b.n_seqs, b.table_stride, b.n_rows};
}

struct RowPlace {
    int seq;    // -1: the row belongs to no sequence
    int pos;
    int rows;   // the sequence's
    int past;
};

// The sequence whose rows hold `row`: row_start does not fall, so it is the number of sequences that end at or before
// it.  64 sequences per load, every lane of the wave takes part; what the place needs is read along with the search.
__device__ inline RowPlace row_place(const PagedSeqs & b, int row, int lane) {
    for (int s0 = 0; s0 < b.n_seqs; s0 += kWave) {
        const int s = min(s0 + lane, b.n_seqs - 1);
        const int start = b.row_start[s], end = b.row_start[s + 1], past = b.n_past[s];
        const uint64_t over = __ballot(s0 + lane >= b.n_seqs || end > row);
        const int l = over != 0 ? __ffsll(static_cast<unsigned long long>(over)) - 1 : kWave;
        if (l == kWave) continue;
        const int first = __builtin_amdgcn_readlane(start, l);
        if (s0 + l >= b.n_seqs || first < 0 || first > row) break;
        const int behind = bounded_past(__builtin_amdgcn_readlane(past, l));
        return RowPlace{s0 + l, behind + row - first, rows_between(first, __builtin_amdgcn_readlane(end, l), b.n_rows), behind};
    }
    return RowPlace{-1, 0, 0, 0};
}

// The rows of one KV head in a paged cache: values of page p from page(p) on, V v_elems behind K, both in elements of CT.  8 bits:
// a page's block ends in its rows' scales, scale(p) is the head's first.
template <typename CT>
struct HeadRows {
    const CT * k;
    int64_t page_elems, v_elems, scales;
    __device__ inline HeadRows(const void * pages, int layer, int n_kv, int n_pages, int page_shift, int head) {
        const int64_t rows = static_cast<int64_t>(1) << page_shift;
        page_elems = n_kv * rows * (sizeof(CT) == 1 ? kQ8RowBytes : kHeadDim);
        v_elems = n_pages * page_elems;
        k = static_cast<const CT *>(pages) + 2 * layer * v_elems + head * rows * kHeadDim;
        scales = n_kv * rows * kHeadDim - head * rows * (kHeadDim - 4);   // from the head's values to its scales, in bytes
    }
    __device__ inline const CT * page(int page) const { return k + page * page_elems; }
    __device__ inline const float * scale(int page) const { return reinterpret_cast<const float *>(k + page * page_elems + scales); }
};

}  // namespace qa
