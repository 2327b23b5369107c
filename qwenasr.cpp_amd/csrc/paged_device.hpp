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
    int seq;   // -1: the row belongs to no sequence
    int pos;
};

// The sequence whose rows hold `row`: row_start does not fall, so it is the number of sequences that end at or before
// it.  64 sequences per load, every lane of the wave takes part.
__device__ inline RowPlace row_place(const PagedSeqs & b, int row, int lane) {
    int seq = 0;
    for (int s0 = 0; s0 < b.n_seqs; s0 += kWave) {
        const int s = s0 + lane;
        const int end = s < b.n_seqs ? b.row_start[s + 1] : row + 1;
        const int n = __popcll(__ballot(end <= row));
        seq += n;
        if (n < kWave) break;
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    if (seq >= b.n_seqs) return RowPlace{-1, 0};
    const int start = b.row_start[seq];
    if (start < 0 || start > row) return RowPlace{-1, 0};
    return RowPlace{seq, bounded_past(b.n_past[seq]) + row - start};
}

}  // namespace qa
