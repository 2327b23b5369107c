// A K/V cache in pages: what its kernels share.
//
// A paged cache is a qa_kv_layout whose streams are pages (n_streams pages of max_seq positions), so one (layer, K or V,
// page) block is [n_kv_heads][positions][head_dim] and every address is cache_row_offset's.  A sequence's table row
// lists its pages in order of position.  Everything that comes from device memory (page numbers, lengths, row starts) is
// bounded here before it becomes an address: a page number outside [0, n_pages) is no page, a position outside the table
// row is no position, a row outside [0, n_rows) is no row.
#pragma once

#include "common.hpp"

namespace qa {

constexpr int kPageMin = 16, kPageMax = 256;   // positions per page: a power of two
constexpr int kMaxCapacity = 1 << 30;          // table_stride * positions per page
constexpr int kMaxGroup = 16;                  // query heads per KV head

// The page of position pos, or -1 where there is none.
__host__ __device__ inline int page_of(const int32_t * table, int table_stride, int page_shift, int n_pages, int pos) {
    const int j = pos >> page_shift;
    if (pos < 0 || j >= table_stride) return -1;
    const int page = table[j];
    return page >= 0 && page < n_pages ? page : -1;
}

// Device memory holds any n_past; positions past 2^30 exist in no table.
__host__ __device__ inline int bounded_past(int n_past) {
    return n_past > kMaxCapacity ? kMaxCapacity : n_past < -kMaxCapacity ? -kMaxCapacity : n_past;
}

// Rows [start, end) of a sequence, cut to the rows that there are.
__host__ __device__ inline int rows_between(int start, int end, int n_rows) {
    if (start < 0) return 0;
    if (end > n_rows) end = n_rows;
    return end > start ? end - start : 0;
}

inline int page_shift_of(int positions) {
    int s = 0;
    while ((1 << s) < positions) ++s;
    return s;
}

inline int check_pages(const qa_kv_layout * l, const char * who) {
    if (qa_kv_layout_check(l) != QA_OK) return QA_ERR_INVALID;
    if (l->head_dim != kHeadDim) return fail(QA_ERR_INVALID, std::string(who) + ": only head_dim 128");
    if (l->max_seq < kPageMin || l->max_seq > kPageMax || (l->max_seq & (l->max_seq - 1)) != 0) {
        return fail(QA_ERR_INVALID, std::string(who) + ": pages of 16, 32, 64, 128 or 256 positions");
    }
    return QA_OK;
}

inline int check_table(int32_t n_rows, int32_t stride, int32_t positions, const char * who) {
    if (n_rows <= 0 || stride <= 0 || static_cast<int64_t>(stride) * positions > kMaxCapacity) {
        return fail(QA_ERR_INVALID, std::string(who) + ": invalid page table");
    }
    return QA_OK;
}

inline int check_batch_sizes(const qa_kv_layout * l, int32_t layer, const qa_paged_batch * b, int32_t n_heads, const char * who) {
    if (check_pages(l, who) != QA_OK) return QA_ERR_INVALID;
    if (!b) return fail(QA_ERR_INVALID, std::string(who) + ": null batch");
    if (layer < 0 || layer >= l->n_layers) return fail(QA_ERR_INVALID, std::string(who) + ": layer out of range");
    if (n_heads <= 0 || n_heads % l->n_kv_heads != 0 || n_heads / l->n_kv_heads > kMaxGroup) {
        return fail(QA_ERR_INVALID, std::string(who) + ": 1 to 16 query heads per KV head");
    }
    if (check_table(b->n_seqs, b->table_stride, l->max_seq, who) != QA_OK) return QA_ERR_INVALID;
    if (b->n_rows < 0 || b->n_rows >= kMaxCapacity || b->max_tokens < 0 || b->max_len < 0) {
        return fail(QA_ERR_INVALID, std::string(who) + ": row, token or position count out of range");
    }
    return QA_OK;
}

inline int check_batch(const qa_kv_layout * l, int32_t layer, const qa_paged_batch * b, int32_t n_heads, const char * who) {
    if (check_batch_sizes(l, layer, b, n_heads, who) != QA_OK) return QA_ERR_INVALID;
    if (b->n_rows > 0 && (!b->tables || !b->n_past || !b->row_start)) {
        return fail(QA_ERR_INVALID, std::string(who) + ": null pointer");
    }
    return QA_OK;
}

// Trees of drafted tokens: mask_words words per row, and rows that 32 bits count in any of their arrays.
constexpr int kMaxMaskWords = 32, kMaxTreeRows = 1 << 24;
inline int check_tree(const qa_paged_batch * b, int32_t mask_words, const char * who) {
    if (!b) return fail(QA_ERR_INVALID, std::string(who) + ": null batch");
    if (b->n_seqs <= 0 || b->n_rows < 0 || b->n_rows > kMaxTreeRows) return fail(QA_ERR_INVALID, std::string(who) + ": row count out of range");
    if (mask_words < 1 || mask_words > kMaxMaskWords) return fail(QA_ERR_INVALID, std::string(who) + ": 1 to 32 words of mask");
    return QA_OK;
}

// Launches go to the current device: a stream of another one is refused before anything is enqueued.
inline int check_stream(void * stream, const char * who) {
    if (!as_stream(stream)) return QA_OK;
    int current = 0;
    hipDevice_t owner = 0;
    if (hipGetDevice(&current) != hipSuccess || hipStreamGetDevice(as_stream(stream), &owner) != hipSuccess) {
        (void)hipGetLastError();
        return fail(QA_ERR_DEVICE, std::string(who) + ": no device behind the stream");
    }
    if (owner != current) return fail(QA_ERR_INVALID, std::string(who) + ": the stream belongs to another device than the current one");
    return QA_OK;
}

}  // namespace qa
