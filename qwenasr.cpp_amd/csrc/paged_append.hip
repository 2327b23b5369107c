// qa_kv_append for a ragged batch over a cache in pages: RMSNorm and RoPE of q and k, and the K/V rows written into the
// page of their position.
//
// One workgroup per token row, one wavefront per head slot at a time, lane i holding elements i and i + 64 (a NEOX
// rotation pair), as in kv_append.hip and through the same norm_rope_pair_cs, so q and the cached rows are the same bits.
// The angles' sine and cosine in 64 bits are as many instructions as a wave's norms: the first wave computes them for all
// four.  (A wave per row, which computes them once without LDS, walks the row's 32 slots alone: 12 instead of 5 us for few
// rows and no faster for 4000.)  The row finds its sequence by a search of row_start in one or two loads; the loads of
// the row do not wait for it.
#include "ops.hpp"
#include "paged.hpp"
#include "paged_device.hpp"
#include "prep.hpp"

namespace qa {
namespace {

struct PagedAppendParams {
    const float * qkv;
    const float * q_norm_w;
    const float * k_norm_w;
    float * q_out;
    void * pages;
    PagedSeqs seqs;
    int32_t n_heads, n_kv_heads, n_pages, page_shift, layer;
    float eps;
};

// STREAM: results past the caches (a prompt of kStreamRows tokens or more): 3913 tokens 23.1 instead of 28.4 us, 1024 tokens 9.3
// instead of 10.4, and the attention that reads them next takes as long.  Fewer results stay in L2 for it (156 tokens with their
// attention 13.3 us, 13.5 past the caches).
constexpr int kStreamRows = 1024;

template <bool STREAM, typename T>
__device__ inline void store_result(T * at, T v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, at);
    else *at = v;
}

template <typename CT, bool STREAM>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendParams p, RopeTable rope) {
#pragma clang fp contract(off)
    __shared__ float s_cos[kHeadDim / 2], s_sin[kHeadDim / 2];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x;
    const int slots = p.n_heads + 2 * p.n_kv_heads;
    const float * src = p.qkv + static_cast<int64_t>(row) * slots * kHeadDim;
    constexpr int kPer = 8;
    float a[kPer], b[kPer];
    auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int slot = min(s0 + 4 * u, slots - 1);   // past the last slot: read again, not stored
            a[u] = src[slot * kHeadDim + lane];
            b[u] = src[slot * kHeadDim + lane + 64];
        }
    };
    load(wave);
    const float wqa = p.q_norm_w[lane], wqb = p.q_norm_w[lane + 64];
    const float wka = p.k_norm_w[lane], wkb = p.k_norm_w[lane + 64];

    const RowPlace at = row_place(p.seqs, row, lane);
    if (at.seq < 0) return;                                // no sequence's row: left as it was
    const int page = page_of(p.seqs.tables + static_cast<int64_t>(at.seq) * p.seqs.table_stride, p.seqs.table_stride,
                             p.page_shift, p.n_pages, at.pos);
    const int slot_in_page = at.pos & ((1 << p.page_shift) - 1);
    float c, s;
    if (wave == 0) {
        rope_cos_sin(at.pos, rope.inv_freq[lane], c, s);
        s_cos[lane] = c;
        s_sin[lane] = s;
    }
    __syncthreads();
    c = s_cos[lane];
    s = s_sin[lane];
    for (int s0 = wave;; s0 += 4 * kPer) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int slot = s0 + 4 * u;
            if (slot >= slots) break;                      // uniform for the wave
            float ra = a[u], rb = b[u];
            if (slot < p.n_heads + p.n_kv_heads) {
                const bool is_q = slot < p.n_heads;
                norm_rope_pair_cs(ra, rb, is_q ? wqa : wka, is_q ? wqb : wkb, p.eps, c, s);
                if (is_q) {
                    float * dst = p.q_out + (static_cast<int64_t>(row) * p.n_heads + slot) * kHeadDim;
                    store_result<STREAM>(dst + lane, ra);
                    store_result<STREAM>(dst + lane + 64, rb);
                    continue;
                }
            }
            if (page < 0) continue;                        // no page holds the position
            const bool is_v = slot >= p.n_heads + p.n_kv_heads;
            const int head = slot - p.n_heads - (is_v ? p.n_kv_heads : 0);
            CT * dst = static_cast<CT *>(p.pages) + cache_row_offset(p.layer, is_v ? 1 : 0, page, head, slot_in_page, p.n_pages,
                                                                     p.n_kv_heads, 1 << p.page_shift);
            store_result<STREAM>(dst + lane, static_cast<CT>(ra));   // f16: rounded to nearest even, the cache's type
            store_result<STREAM>(dst + lane + 64, static_cast<CT>(rb));
        }
        if (s0 + 4 * kPer >= slots) break;
        load(s0 + 4 * kPer);
    }
}

}  // namespace
}  // namespace qa

extern "C" int qa_paged_append(const float * qkv, const float * q_norm_w, const float * k_norm_w, float * q_out, void * pages,
                               const qa_kv_layout * layout, int32_t layer, const qa_paged_batch * batch, int32_t n_heads,
                               float rope_theta, float eps, void * stream) {
    using namespace qa;
    if (check_batch(layout, layer, batch, n_heads, "qa_paged_append") != QA_OK) return QA_ERR_INVALID;
    if (!(rope_theta > 0.0f)) return fail(QA_ERR_INVALID, "qa_paged_append: rope_theta must be positive");
    if (batch->n_rows == 0) return QA_OK;
    if (!qkv || !q_norm_w || !k_norm_w || !q_out || !pages) return fail(QA_ERR_INVALID, "qa_paged_append: null pointer");
    if (const int rc = check_stream(stream, "qa_paged_append"); rc != QA_OK) return rc;
    PagedAppendParams p{};
    p.qkv = qkv;
    p.q_norm_w = q_norm_w;
    p.k_norm_w = k_norm_w;
    p.q_out = q_out;
    p.pages = pages;
    p.seqs = paged_seqs(*batch);
    p.n_heads = n_heads;
    p.n_kv_heads = layout->n_kv_heads;
    p.n_pages = layout->n_streams;
    p.page_shift = page_shift_of(layout->max_seq);
    p.layer = layer;
    p.eps = eps;
    const RopeTable rope = make_rope_table(rope_theta);
    const dim3 grid(static_cast<unsigned>(batch->n_rows));
    const bool stream_out = batch->n_rows >= kStreamRows;
    const auto f16 = stream_out ? &paged_append_kernel<_Float16, true> : &paged_append_kernel<_Float16, false>;
    const auto f32 = stream_out ? &paged_append_kernel<float, true> : &paged_append_kernel<float, false>;
    const auto kernel = layout->cache_type == QA_CACHE_F16 ? f16 : f32;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, as_stream(stream), p, rope);
    QA_LAUNCH_CHECK("paged_append_kernel");
    return QA_OK;
}
