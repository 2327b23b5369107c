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

#include <type_traits>

namespace qa {
namespace {

struct PagedAppendParams {
    const float * qkv;
    const float * q_norm_w;
    const float * k_norm_w;
    float * q_out;
    void * pages;
    PagedSeqs seqs;
    const int32_t * depth;   // null, or what a row's angle has in the place of its number in the sequence
    int32_t n_heads, n_kv_heads, n_pages, page_shift, layer;
    float eps;
};

// A row of 128 values in 8 bits, lane holding a and b: the integers nearest to x / scale, scale = max |x| / 127.  A prompt's append
// is bound by its instructions, so the quotients are products with a reciprocal and a correction, which rounds them as a
// division does, integers come from the low bits of 1.5 2^23 + x, and four lanes put a word together.  Scales that are no ordinary
// numbers take the divisions.  3913 rows of 16 query and 8 KV heads 26.3 us, 104 MB at 4.0 TB/s (f16 22.4, 112 MB at 5.0; a copy
// reaches 5.1); 32 rows 4.6.
struct Q8Row {
    uint32_t a, b;      // the byte at its place in the word of four lanes
    float scale;
};

__device__ inline Q8Row quantised(float a, float b, uint32_t place) {
    // as integers infinities and NaN are the largest
    uint32_t most = max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu);
#pragma unroll
    for (int step = 0; step < 6; ++step) {
        const uint32_t o = step == 0 ? __builtin_amdgcn_mov_dpp(most, 0xB1, 0xf, 0xf, false) : step == 1 ? __builtin_amdgcn_mov_dpp(most, 0x4E, 0xf, 0xf, false)
                         : step == 2 ? __builtin_amdgcn_mov_dpp(most, 0x141, 0xf, 0xf, false) : step == 3 ? __builtin_amdgcn_mov_dpp(most, 0x140, 0xf, 0xf, false)
                         : step == 4 ? __builtin_amdgcn_update_dpp(0, most, 0x142, 0xa, 0xf, false) : __builtin_amdgcn_update_dpp(0, most, 0x143, 0xc, 0xf, false);
        most = max(most, o);
    }
    most = __builtin_amdgcn_readlane(most, 63);
    const float mx = __uint_as_float(most);
    float scale, qa, qb;
    if (mx > 1e-25f && mx < 1e35f) {
        constexpr float kPart = 1.0f / 127.0f;
        scale = mx * kPart;
        scale = fmaf(fmaf(-scale, 127.0f, mx), kPart, scale);
        float r = __builtin_amdgcn_rcpf(scale);
        r = fmaf(fmaf(-scale, r, 1.0f), r, r);
        qa = a * r;
        qb = b * r;
        qa = fmaf(fmaf(-qa, scale, a), r, qa);
        qb = fmaf(fmaf(-qb, scale, b), r, qb);
    } else {
        if (most >= 0x7f800000u) return Q8Row{0, 0, NAN};
        scale = mx / 127.0f;
        // a scale that rounds among the smallest numbers may leave more than 127 of them
        qa = scale > 0.0f ? fminf(fmaxf(a / scale, -127.0f), 127.0f) : 0.0f;
        qb = scale > 0.0f ? fminf(fmaxf(b / scale, -127.0f), 127.0f) : 0.0f;
    }
    constexpr float kWhole = 12582912.0f;
    return Q8Row{__builtin_amdgcn_perm(0u, __float_as_uint(qa + kWhole), place), __builtin_amdgcn_perm(0u, __float_as_uint(qb + kWhole), place), scale};
}

// Four lanes' bytes in one word, the same in all four.
__device__ inline uint32_t quad_word(uint32_t w) {
    w |= __builtin_amdgcn_mov_dpp(w, 0xB1, 0xf, 0xf, false);
    w |= __builtin_amdgcn_mov_dpp(w, 0x4E, 0xf, 0xf, false);
    return w;
}

// STREAM: results past the caches (a prompt of kStreamRows tokens or more).  Six layers' inputs in turn, f16: 1024 tokens 8.9 instead of
// 9.6 us, 2000 13.5 / 15.4, 3913 26.4 / 28.0 (f32 pages 9.1 / 10.2, 13.7 / 17.8, 27.9 / 30.5), and the attention that reads them next takes as
// long.  Fewer results stay in L2 for it (156 tokens with their attention 13.3 us, 13.5 past the caches).
constexpr int kStreamRows = 1024;
// Waves per row: a wave walks its head slots one after another, which few rows wait for (32 rows of f16 in 4 / 8 / 16 waves 5.2 / 4.6 /
// 4.6 us); of many rows each wave's angles and place are more to do.
constexpr int append_waves(bool stream) { return stream ? 4 : 8; }
constexpr int append_threads(bool stream) { return append_waves(stream) * kWave; }

template <bool STREAM, typename T>
__device__ inline void store_result(T * at, T v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, at);
    else *at = v;
}

template <typename CT, bool STREAM>
__global__ __launch_bounds__(append_threads(STREAM)) void paged_append_kernel(PagedAppendParams p, RopeTable rope) {
#pragma clang fp contract(off)
    __shared__ float s_cos[kHeadDim / 2], s_sin[kHeadDim / 2];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x;
    const int slots = p.n_heads + 2 * p.n_kv_heads;
    const float * src = p.qkv + static_cast<int64_t>(row) * slots * kHeadDim;
    constexpr int W = append_waves(STREAM), kPer = 32 / W;   // slots in flight: those of 16 query and 8 KV heads
    float a[kPer], b[kPer];
    auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int slot = min(s0 + W * u, slots - 1);   // past the last slot: read again, not stored
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
        // any depth: the sum wraps, as no pointer depends on it
        const int turn = p.depth ? static_cast<int>(static_cast<uint32_t>(at.past) + static_cast<uint32_t>(p.depth[row])) : at.pos;
        rope_cos_sin(turn, rope.inv_freq[lane], c, s);
        s_cos[lane] = c;
        s_sin[lane] = s;
    }
    __syncthreads();
    c = s_cos[lane];
    s = s_sin[lane];
    for (int s0 = wave;; s0 += W * kPer) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int slot = s0 + W * u;
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
            if constexpr (std::is_same<CT, int8_t>::value) {
                const HeadRows<int8_t> rows(p.pages, p.layer, p.n_kv_heads, p.n_pages, p.page_shift, head);
                const int64_t v = is_v ? rows.v_elems : 0;
                int8_t * dst = const_cast<int8_t *>(rows.page(page)) + v + slot_in_page * kHeadDim;
                // byte 0 of the source goes to byte lane % 4, the others are zeros (selector 12)
                const uint32_t place = 0x0c0c0c0cu ^ (0x0cu << ((lane & 3) * 8));
                const Q8Row r = quantised(ra, rb, place);
                // 32 lanes store 4 bytes each: the first of four lanes the lower half's, the second the upper half's
                const uint32_t lower = quad_word(r.a), upper = quad_word(r.b);
                if ((lane & 2) == 0) store_result<STREAM>(reinterpret_cast<uint32_t *>(dst + (lane & ~3) + (lane & 1) * 64), lane & 1 ? upper : lower);
                if (lane == 0) const_cast<float *>(rows.scale(page))[v / 4 + slot_in_page] = r.scale;
            } else {
                CT * dst = static_cast<CT *>(p.pages) + cache_row_offset(p.layer, is_v ? 1 : 0, page, head, slot_in_page, p.n_pages,
                                                                         p.n_kv_heads, 1 << p.page_shift);
                store_result<STREAM>(dst + lane, static_cast<CT>(ra));   // f16: rounded to nearest even, the cache's type
                store_result<STREAM>(dst + lane + 64, static_cast<CT>(rb));
            }
        }
        if (s0 + W * kPer >= slots) break;
        load(s0 + W * kPer);
    }
}

// 8 consecutive values per lane and load.  Many rows: a wave per row, four loads in flight behind the row's place (a workgroup
// per row waited for that place twice as often: 3913 rows of 8 bits as f16 9.5 us, so 7.2).  Few rows: a workgroup per row.
constexpr int kReadUnits = kHeadDim / 8;

struct PagedReadParams {
    const void * pages;
    void * out[2];
    PagedSeqs seqs;
    int32_t n_kv_heads, n_pages, page_shift, layer;
};

template <typename CT, typename OT, int WAVES>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedReadParams p) {
    constexpr int kLoads = 4 / WAVES;
    typedef CT in8 __attribute__((ext_vector_type(8), aligned(sizeof(CT) == 1 ? 8 : 16)));
    typedef OT out8 __attribute__((ext_vector_type(8), aligned(16)));
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x * kLoads + wave / WAVES;
    if (row >= p.seqs.n_rows) return;
    const RowPlace at = row_place(p.seqs, row, lane);
    if (at.seq < 0) return;
    const int page = page_of(p.seqs.tables + static_cast<int64_t>(at.seq) * p.seqs.table_stride, p.seqs.table_stride,
                             p.page_shift, p.n_pages, at.pos);
    const int slot = at.pos & ((1 << p.page_shift) - 1);
    const int units = p.n_kv_heads * kReadUnits;                       // of K, and of V
    for (int first = wave % WAVES * kWave + lane; first < 2 * units; first += 4 * kWave) {
        in8 x[kLoads];
        float scale[kLoads];
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const int u = min(first + k * WAVES * kWave, 2 * units - 1), kv = u >= units ? 1 : 0, unit = u - kv * units;
            const HeadRows<CT> rows(p.pages, p.layer, p.n_kv_heads, p.n_pages, p.page_shift, unit / kReadUnits);
            const int64_t behind = kv ? rows.v_elems : 0;
            // without a page: page 0, which there always is, and not used
            x[k] = *reinterpret_cast<const in8 *>(rows.page(max(page, 0)) + behind + slot * kHeadDim + unit % kReadUnits * 8);
            if constexpr (std::is_same<CT, int8_t>::value) scale[k] = rows.scale(max(page, 0))[behind / 4 + slot];
        }
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const int u = first + k * WAVES * kWave, kv = u >= units ? 1 : 0;
            if (u >= 2 * units || !p.out[kv]) continue;
            out8 v = {};
            if (page >= 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (std::is_same<CT, int8_t>::value) {
                        float f = static_cast<float>(x[k][e]) * scale[k];
                        asm("" : "+v"(f));                 // the f32 that a reader of f32 gets, rounded to f16, and not the product
                        v[e] = static_cast<OT>(f);
                    } else {
                        v[e] = static_cast<OT>(x[k][e]);
                    }
                }
            }
            *reinterpret_cast<out8 *>(static_cast<OT *>(p.out[kv]) + (static_cast<int64_t>(row) * units + u - kv * units) * 8) = v;
        }
    }
}

template <typename CT, typename OT>
void launch_read(const PagedReadParams & p, hipStream_t stream) {
    const bool many = p.seqs.n_rows >= kStreamRows;
    const auto kernel = many ? &paged_read_kernel<CT, OT, 1> : &paged_read_kernel<CT, OT, 4>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(many ? (p.seqs.n_rows + 3) / 4 : p.seqs.n_rows)), dim3(256), 0, stream, p);
}

template <typename CT>
void launch_read(const PagedReadParams & p, int32_t out_type, hipStream_t stream) {
    if (out_type == QA_CACHE_F16) launch_read<CT, _Float16>(p, stream);
    else launch_read<CT, float>(p, stream);
}

int append(const float * qkv, const float * q_norm_w, const float * k_norm_w, float * q_out, void * pages, const qa_kv_layout * layout,
           int32_t layer, const qa_paged_batch * batch, const int32_t * depth, int32_t n_heads, float rope_theta, float eps,
           void * stream, const char * name) {
    const std::string who = name;
    if (check_batch(layout, layer, batch, n_heads, name) != QA_OK) return QA_ERR_INVALID;
    if (!(rope_theta > 0.0f)) return fail(QA_ERR_INVALID, who + ": rope_theta must be positive");
    if (batch->n_rows == 0) return QA_OK;
    if (!qkv || !q_norm_w || !k_norm_w || !q_out || !pages) return fail(QA_ERR_INVALID, who + ": null pointer");
    // 8 bits are stored in words, and their scales as f32
    if (layout->cache_type == QA_CACHE_Q8 && (reinterpret_cast<uintptr_t>(pages) & 15) != 0) {
        return fail(QA_ERR_INVALID, who + ": pages must be aligned to 16 bytes");
    }
    if (const int rc = check_stream(stream, name); rc != QA_OK) return rc;
    PagedAppendParams p{};
    p.qkv = qkv;
    p.q_norm_w = q_norm_w;
    p.k_norm_w = k_norm_w;
    p.q_out = q_out;
    p.pages = pages;
    p.seqs = paged_seqs(*batch);
    p.depth = depth;
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
    const auto q8 = stream_out ? &paged_append_kernel<int8_t, true> : &paged_append_kernel<int8_t, false>;
    const auto kernel = layout->cache_type == QA_CACHE_Q8 ? q8 : layout->cache_type == QA_CACHE_F16 ? f16 : f32;
    hipLaunchKernelGGL(kernel, grid, dim3(append_threads(stream_out)), 0, as_stream(stream), p, rope);
    QA_LAUNCH_CHECK("paged_append_kernel");
    return QA_OK;
}

}  // namespace
}  // namespace qa

extern "C" int qa_paged_append(const float * qkv, const float * q_norm_w, const float * k_norm_w, float * q_out, void * pages,
                               const qa_kv_layout * layout, int32_t layer, const qa_paged_batch * batch, int32_t n_heads,
                               float rope_theta, float eps, void * stream) {
    return qa::append(qkv, q_norm_w, k_norm_w, q_out, pages, layout, layer, batch, nullptr, n_heads, rope_theta, eps, stream,
                      "qa_paged_append");
}

extern "C" int qa_paged_tree_append(const float * qkv, const float * q_norm_w, const float * k_norm_w, float * q_out, void * pages,
                                    const qa_kv_layout * layout, int32_t layer, const qa_paged_batch * batch, const int32_t * depth,
                                    int32_t n_heads, float rope_theta, float eps, void * stream) {
    if (batch && batch->n_rows > 0 && !depth) return qa::fail(QA_ERR_INVALID, "qa_paged_tree_append: null pointer");
    return qa::append(qkv, q_norm_w, k_norm_w, q_out, pages, layout, layer, batch, depth, n_heads, rope_theta, eps, stream,
                      "qa_paged_tree_append");
}

extern "C" int qa_paged_read(const void * pages, const qa_kv_layout * layout, int32_t layer, const qa_paged_batch * batch, void * k_out,
                             void * v_out, int32_t out_type, void * stream) {
    using namespace qa;
    const char * who = "qa_paged_read";
    if (check_batch(layout, layer, batch, layout ? layout->n_kv_heads : 0, who) != QA_OK) return QA_ERR_INVALID;
    if (out_type != QA_CACHE_F32 && out_type != QA_CACHE_F16) return fail(QA_ERR_INVALID, "qa_paged_read: rows of f32 or f16");
    if (batch->n_rows == 0 || (!k_out && !v_out)) return QA_OK;
    if (!pages) return fail(QA_ERR_INVALID, "qa_paged_read: null pointer");
    if (((reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) != 0) {
        return fail(QA_ERR_INVALID, "qa_paged_read: pointers must be aligned to 16 bytes");
    }
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    PagedReadParams p{};
    p.pages = pages;
    p.out[0] = k_out;
    p.out[1] = v_out;
    p.seqs = paged_seqs(*batch);
    p.n_kv_heads = layout->n_kv_heads;
    p.n_pages = layout->n_streams;
    p.page_shift = page_shift_of(layout->max_seq);
    p.layer = layer;
    if (layout->cache_type == QA_CACHE_Q8) launch_read<int8_t>(p, out_type, as_stream(stream));
    else if (layout->cache_type == QA_CACHE_F16) launch_read<_Float16>(p, out_type, as_stream(stream));
    else launch_read<float>(p, out_type, as_stream(stream));
    QA_LAUNCH_CHECK("paged_read_kernel");
    return QA_OK;
}
