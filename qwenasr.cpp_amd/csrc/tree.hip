// Trees of drafted tokens over a cache in pages: masks and depths, the path that a step accepts, and its rows moved together.
//
// A tree is a few dozen nodes, so the first two cost their dependent loads: a workgroup per sequence reads the parents into
// LDS at once, and every walk is LDS reads.  A parent has a lower number than its child, so walks end, a path's nodes rise, and
// a row's mask is written from its highest word down while its ancestors are passed.  8 nodes take 1.8 us each, sixteen trees of up to
// 41 nodes 3.2 and 2.9, most of it the launch and two levels of loads.
#include "common.hpp"
#include "paged.hpp"
#include "paged_device.hpp"

#include <algorithm>

namespace qa {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kTreeThreads = 256;
constexpr int kMaxNodes = 32 * kMaxMaskWords;   // rows of a sequence behind them belong to no tree

// The nodes of sequence s: its first row, and how many.
__device__ inline int nodes_of(const PagedSeqs & b, int s, int & first) {
    first = b.row_start[s];
    return min(rows_between(first, b.row_start[s + 1], b.n_rows), kMaxNodes);
}

__global__ __launch_bounds__(kTreeThreads) void tree_prepare_kernel(PagedSeqs seqs, const int32_t * parents, uint32_t * mask, int mask_words,
                                                                    int32_t * depth) {
    __shared__ int s_parent[kMaxNodes];
    int first;
    const int n = nodes_of(seqs, blockIdx.x, first);
    for (int i = threadIdx.x; i < n; i += kTreeThreads) {
        const int up = parents[first + i];
        s_parent[i] = up >= 0 && up < i ? up : -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kTreeThreads) {
        uint32_t * words = mask + static_cast<int64_t>(first + i) * mask_words;
        int passed = -1, at = mask_words - 1;             // the word that is being filled
        uint32_t bits = 0;
        for (int node = i; node >= 0; node = s_parent[node], ++passed) {
            if ((node >> 5) >= mask_words) continue;
            for (; at > (node >> 5); --at, bits = 0) words[at] = bits;
            bits |= 1u << (node & 31);
        }
        for (; at >= 0; --at, bits = 0) words[at] = bits;
        depth[first + i] = passed;
    }
}

__global__ __launch_bounds__(kTreeThreads) void tree_accept_kernel(PagedSeqs seqs, const int32_t * parents, const int32_t * ids,
                                                                   const int32_t * picks, int32_t * path, int32_t * n_kept, int32_t * next) {
    __shared__ int s_child[kMaxNodes], s_pick[kMaxNodes], s_path[kMaxNodes];
    __shared__ int s_kept;
    int first;
    const int n = nodes_of(seqs, blockIdx.x, first);
    if (n == 0) {
        if (threadIdx.x == 0) {
            n_kept[blockIdx.x] = 0;
            next[blockIdx.x] = -1;
        }
        return;
    }
    constexpr int kPer = kMaxNodes / kTreeThreads;
    int up[kPer], id[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
        const int i = threadIdx.x + u * kTreeThreads;
        if (i >= n) continue;
        up[u] = parents[first + i];
        id[u] = ids[first + i];
        s_pick[i] = picks[first + i];
        s_child[i] = kMaxNodes;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
        const int i = threadIdx.x + u * kTreeThreads;
        if (i < n && up[u] >= 0 && up[u] < i && id[u] == s_pick[up[u]]) atomicMin(&s_child[up[u]], i);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int kept = 0, node = 0, last = 0;
        for (; node < n; node = s_child[node]) s_path[kept++] = last = node;
        s_kept = kept;
        n_kept[blockIdx.x] = kept;
        next[blockIdx.x] = s_pick[last];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kTreeThreads) path[first + i] = i < s_kept ? s_path[i] : -1;
}

struct KeepParams {
    char * pages;
    PagedSeqs seqs;
    const int32_t * path;
    const int32_t * n_kept;
    int64_t block_bytes;     // one (layer, K or V) block of a page
    int32_t row_bytes, n_kv, n_pages, page_shift;
    bool scales;             // 8 bits: rows have a scale each behind the block's values
};

// Workgroup ((layer, K or V), sequence, up to kKeepHeads heads).  A path rises, so node path[k] >= k: rows are taken in order of k,
// as many at a time as the workgroup's registers hold, and all of them are read before one is written.  Then nothing that is
// read later has been written before: it lies at path[j] > path[k] >= k for j > k.  28 layers of 8 heads, f16: 3.5 us for 5 rows of one
// sequence, 5.9 for sixteen sequences' (three levels of dependent loads; their rows are 2 MB).
constexpr int kKeepHeads = 8, kKeepPer = 4, kKeepThreads = 256;

__global__ __launch_bounds__(kKeepThreads) void paged_keep_kernel(KeepParams p) {
    constexpr int kWindow = kMaxNodes / kPageMin + 2;      // table entries of a sequence's nodes
    __shared__ int s_from[kMaxNodes], s_page[kWindow], s_end;
    const int s = blockIdx.y;
    const int head0 = blockIdx.z * kKeepHeads, heads = min(kKeepHeads, p.n_kv - head0);
    if (threadIdx.x == 0) s_end = kMaxNodes;
    __syncthreads();
    // its time is dependent loads: the sequence's numbers, then its path and its table's entries, then rows
    const int past = bounded_past(p.seqs.n_past[s]), asked = p.n_kept[s];
    int first;
    const int nodes = nodes_of(p.seqs, s, first);
    const int kept = min(max(asked, 0), nodes);
    const int32_t * table = p.seqs.tables + static_cast<int64_t>(s) * p.seqs.table_stride;
    const int first_entry = past >> p.page_shift;
    for (int k = threadIdx.x; k < kept; k += kKeepThreads) {
        const int from = p.path[first + k], before = k > 0 ? p.path[first + k - 1] : -1;
        s_from[k] = from;
        if (from <= before || from >= nodes) atomicMin(&s_end, k);
    }
    if (static_cast<int>(threadIdx.x) < kWindow) {
        const int64_t pos = (static_cast<int64_t>(first_entry) + threadIdx.x) << p.page_shift;
        s_page[threadIdx.x] = pos < kMaxCapacity ? page_of(table, p.seqs.table_stride, p.page_shift, p.n_pages, static_cast<int>(pos)) : -1;
    }
    __syncthreads();
    const int n = min(s_end, kept);
    char * base = p.pages + static_cast<int64_t>(blockIdx.x) * p.n_pages * p.block_bytes;
    const int units = p.row_bytes / 16, per_row = heads * units, in_page = (1 << p.page_shift) - 1;
    const int chunk = kKeepPer * kKeepThreads / per_row;   // rows at a time
    // Where the k-th row comes from and goes to, in bytes from base, for rows of `bytes` behind `offset` of a block; false: stays
    auto places = [&](int k, int head, int64_t offset, int bytes, int64_t & from, int64_t & to) {
        const int a = past + s_from[k], b = past + k;
        const int pa = s_page[(a >> p.page_shift) - first_entry], pb = s_page[(b >> p.page_shift) - first_entry];
        if (a == b || pa < 0 || pb < 0) return false;
        from = pa * p.block_bytes + offset + ((static_cast<int64_t>(head) << p.page_shift) + (a & in_page)) * bytes;
        to = pb * p.block_bytes + offset + ((static_cast<int64_t>(head) << p.page_shift) + (b & in_page)) * bytes;
        return true;
    };
    for (int k0 = 0; k0 < n; k0 += chunk) {
        const int rows = min(chunk, n - k0);
        u4 v[kKeepPer];
        int64_t to[kKeepPer];
        float scale = 0.0f;
        int64_t scale_to = -1;
#pragma unroll
        for (int u = 0; u < kKeepPer; ++u) {
            const int item = threadIdx.x + u * kKeepThreads, row = item / per_row, rest = item - row * per_row;
            int64_t from = 0;
            to[u] = -1;
            if (row >= rows || !places(k0 + row, head0 + rest / units, 0, p.row_bytes, from, to[u])) {
                to[u] = -1;
                continue;
            }
            v[u] = *reinterpret_cast<const u4 *>(base + from + rest % units * 16);
            to[u] += rest % units * 16;
        }
        if (p.scales && static_cast<int>(threadIdx.x) < rows * heads) {
            int64_t from = 0;
            const int row = threadIdx.x / heads, head = head0 + threadIdx.x % heads;
            if (places(k0 + row, head, (static_cast<int64_t>(p.n_kv) << p.page_shift) * kHeadDim, 4, from, scale_to)) {
                scale = *reinterpret_cast<const float *>(base + from);
            } else {
                scale_to = -1;
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every row has arrived before any is written over
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kKeepPer; ++u) {
            if (to[u] >= 0) *reinterpret_cast<u4 *>(base + to[u]) = v[u];
        }
        if (scale_to >= 0) *reinterpret_cast<float *>(base + scale_to) = scale;
    }
}

int check_tree_batch(const qa_paged_batch * b, int32_t mask_words, bool pointers, const char * who) {
    if (check_tree(b, mask_words, who) != QA_OK) return QA_ERR_INVALID;
    if (!b->row_start || !pointers) return fail(QA_ERR_INVALID, std::string(who) + ": null pointer");
    return QA_OK;
}

}  // namespace
}  // namespace qa

extern "C" int qa_tree_prepare(const qa_paged_batch * batch, const int32_t * parents, uint32_t * mask, int32_t mask_words,
                               int32_t * depth, void * stream) {
    using namespace qa;
    const char * who = "qa_tree_prepare";
    if (check_tree(batch, mask_words, who) != QA_OK) return QA_ERR_INVALID;
    if (batch->n_rows == 0) return QA_OK;
    if (check_tree_batch(batch, mask_words, parents && mask && depth, who) != QA_OK) return QA_ERR_INVALID;
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    hipLaunchKernelGGL(tree_prepare_kernel, dim3(static_cast<unsigned>(batch->n_seqs)), dim3(kTreeThreads), 0, as_stream(stream),
                       paged_seqs(*batch), parents, mask, mask_words, depth);
    QA_LAUNCH_CHECK("tree_prepare_kernel");
    return QA_OK;
}

extern "C" int qa_tree_accept(const qa_paged_batch * batch, const int32_t * parents, const int32_t * ids, const int32_t * picks,
                              int32_t * path, int32_t * n_kept, int32_t * next, void * stream) {
    using namespace qa;
    const char * who = "qa_tree_accept";
    if (check_tree(batch, 1, who) != QA_OK) return QA_ERR_INVALID;
    const bool rows = batch->n_rows == 0 || (parents && ids && picks && path);   // without rows every sequence keeps none
    if (check_tree_batch(batch, 1, rows && n_kept && next, who) != QA_OK) return QA_ERR_INVALID;
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    hipLaunchKernelGGL(tree_accept_kernel, dim3(static_cast<unsigned>(batch->n_seqs)), dim3(kTreeThreads), 0, as_stream(stream),
                       paged_seqs(*batch), parents, ids, picks, path, n_kept, next);
    QA_LAUNCH_CHECK("tree_accept_kernel");
    return QA_OK;
}

extern "C" int qa_paged_keep(void * pages, const qa_kv_layout * layout, const qa_paged_batch * batch, const int32_t * path,
                             const int32_t * n_kept, void * stream) {
    using namespace qa;
    const char * who = "qa_paged_keep";
    if (check_batch(layout, 0, batch, layout ? layout->n_kv_heads : 0, who) != QA_OK) return QA_ERR_INVALID;
    if (check_tree(batch, 1, who) != QA_OK) return QA_ERR_INVALID;
    if (batch->n_rows == 0) return QA_OK;
    if (!pages || !path || !n_kept) return fail(QA_ERR_INVALID, "qa_paged_keep: null pointer");
    if ((reinterpret_cast<uintptr_t>(pages) & 15) != 0) return fail(QA_ERR_INVALID, "qa_paged_keep: pages must be aligned to 16 bytes");
    const int groups = (layout->n_kv_heads + kKeepHeads - 1) / kKeepHeads;
    if (batch->n_seqs > 65535 || groups > 65535 || layout->n_layers > (1 << 22)) return fail(QA_ERR_INVALID, "qa_paged_keep: more than 65535 sequences");
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    KeepParams p{};
    p.pages = static_cast<char *>(pages);
    p.seqs = paged_seqs(*batch);
    p.path = path;
    p.n_kept = n_kept;
    p.block_bytes = block_bytes(*layout);
    p.row_bytes = static_cast<int32_t>(kHeadDim * qa_kv_elem_bytes(layout->cache_type));
    p.n_kv = layout->n_kv_heads;
    p.n_pages = layout->n_streams;
    p.page_shift = page_shift_of(layout->max_seq);
    p.scales = layout->cache_type == QA_CACHE_Q8;
    const dim3 grid(static_cast<unsigned>(2 * layout->n_layers), static_cast<unsigned>(batch->n_seqs), static_cast<unsigned>(groups));
    hipLaunchKernelGGL(paged_keep_kernel, grid, dim3(kKeepThreads), 0, as_stream(stream), p);
    QA_LAUNCH_CHECK("paged_keep_kernel");
    return QA_OK;
}
