// Matrix-vector products with 4-bit weights: y = W x for 1 to 32 token rows, w = (q - 8) d, q in 0..15, d an f16 scale per
// row and group of 32, 64 or 128 columns, with the RMSNorm before and the SwiGLU behind that the decoder's GEMVs fuse.
//
// What bounds it is the stream of W: half a byte per weight, 1/8 of the f32 GEMV's.  A block of 16 rows x 128 columns is
// 1 KB, one 16-byte load per lane, and lies in the order in which v_mfma_f32_16x16x32_f16 takes it as its A operand: lane
// 16 j + r holds row r, and its word w the columns 32 w + 8 j .. + 7, so no weight moves between lanes.  Nibbles become
// f16 by bit operations: 0x6400 | q is 1024 + q, and a packed add takes 1032 off.  q - 8 is exact in f16.
//
// x is f32.  It is split into two f16 parts (a power of two per row brings the largest finite |x| to 2^14..2^15), which
// stand side by side in the 16 columns of the B operand: 8 rows in one product, so that a single row costs no more
// matrix instructions than eight.  Products are exact in f32, what the split leaves out is 2^-22 of a value (or 2^-39 of the
// row's largest, where that is more), a group's sum
// is multiplied by its scale in f32 and added up in f32.
#include "ops.hpp"
#include "paged.hpp"
#include "wave.hpp"

#include <algorithm>

namespace qa {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16, kTileCols = 128;
constexpr int kQ4MaxRows = 32;
constexpr int kQ4Waves = 8;                        // per workgroup
constexpr int kQ4Threads = kQ4Waves * kWave;
constexpr int kXBytes = 64 * 1024;                 // of x in LDS at a time: two workgroups per CU
constexpr int kQ4Exp = 15;                        // a row's largest finite |x| goes to [2^14, 2^15)

struct Q4Params {
    const uint8_t * W;
    const _Float16 * scales;
    const float * x;
    float * y;
    const float * norm_w;
    int32_t out_dim, in_dim, rows, group_shift;   // group = 32 << group_shift
    int32_t n_tiles, tile_up;                     // tiles of y, and the distance to a tile's up rows
    int32_t wt, wk;                               // waves over tiles and over columns: wt * wk = kQ4Waves
    int32_t chunk;                                // columns of x in LDS at a time
    int32_t epilogue;
    float eps;
};

// 8 nibbles of a word as q - 8 in f16, in column order: column e lies in bits 4 (e / 2) + 16 (e % 2).
__device__ inline h8 unpack(uint32_t w) {
    const h2 off = h2{static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
    h8 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const h2 v = __builtin_bit_cast(h2, ((w >> (4 * e)) & 0x000f000fu) | 0x64006400u) + off;
        r[2 * e] = v[0];
        r[2 * e + 1] = v[1];
    }
    return r;
}

// NB: blocks of 8 x rows.  TW: tiles per wave whose blocks are in flight together (2 with SwiGLU: gate and up).
template <int NB, int TW, bool SWIGLU>
__global__ __launch_bounds__(kQ4Threads, 2) void gemv_q4_kernel(Q4Params p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    _Float16 * sx = reinterpret_cast<_Float16 *>(lds);            // [chunk / 32][2 rows][32]
    __shared__ float s_scale[kQ4MaxRows];                         // RMSNorm factor of each row
    __shared__ int s_exp[kQ4MaxRows];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    const int wk = wave % p.wk, wt = wave / p.wk;
    const int tile0 = (static_cast<int>(blockIdx.x) * p.wt + wt) * (SWIGLU ? 1 : TW);
    const int n_kb = p.in_dim / kTileCols;

    // the factor of each x row: RMSNorm and the power of two of the split
    for (int r = wave; r < p.rows; r += kQ4Waves) {
        const float * x = p.x + static_cast<int64_t>(r) * p.in_dim;
        double ss = 0.0;
        float mx = 0.0f;
        for (int k = lane; k < p.in_dim; k += kWave) {
            const float v = x[k];
            ss += static_cast<double>(v) * v;
            const float a = fabsf(p.norm_w ? v * p.norm_w[k] : v);
            if (a < INFINITY) mx = fmaxf(mx, a);                  // what is not finite passes through hi as it is
        }
        const float f = p.norm_w ? 1.0f / sqrtf(static_cast<float>(wave_sum_d_all(ss) / p.in_dim) + p.eps) : 1.0f;
        mx = wave_max_all(mx) * f;
        if (lane == 0) {
            s_scale[r] = f;
            s_exp[r] = mx > 0.0f && mx < INFINITY ? kQ4Exp - __builtin_amdgcn_frexp_expf(mx) : 0;
        }
    }

    const u4 * wp[TW];
    const _Float16 * dp[TW];
    const int n_groups = p.in_dim >> (5 + p.group_shift);
#pragma unroll
    for (int t = 0; t < TW; ++t) {
        // tiles behind the last one read it again and store nothing
        const int tile = SWIGLU ? min(tile0, p.n_tiles - 1) + t * p.tile_up : min(tile0 + t, p.n_tiles - 1);
        wp[t] = reinterpret_cast<const u4 *>(p.W) + static_cast<int64_t>(tile) * n_kb * kWave + lane;
        dp[t] = p.scales + static_cast<int64_t>(tile) * n_groups * kTileRows + g4 * 4;
    }
    f4 acc[TW][NB];
#pragma unroll
    for (int t = 0; t < TW; ++t) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[t][nb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int cols = 2 * p.rows;
    int bcol[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) bcol[nb] = 2 * min(nb * 8 + (c16 & 7), p.rows - 1) + (c16 >> 3);

    u4 w[TW], w_next[TW];
    int kb = wk;
#pragma unroll
    for (int t = 0; t < TW; ++t) w_next[t] = wp[t][static_cast<int64_t>(min(kb, n_kb - 1)) * kWave];
    for (int k0 = 0; k0 < p.in_dim; k0 += p.chunk) {
        const int k1 = min(k0 + p.chunk, p.in_dim);
        __syncthreads();
        for (int idx = threadIdx.x; idx < p.rows * ((k1 - k0) >> 2); idx += kQ4Threads) {
            const int r = idx / ((k1 - k0) >> 2), k = k0 + (idx - r * ((k1 - k0) >> 2)) * 4;
            f4 v = *reinterpret_cast<const f4 *>(p.x + static_cast<int64_t>(r) * p.in_dim + k);
            if (p.norm_w) v = v * s_scale[r] * *reinterpret_cast<const f4 *>(p.norm_w + k);
            h4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float s = ldexpf(v[e], s_exp[r]);
                hi[e] = static_cast<_Float16>(s);
                lo[e] = static_cast<_Float16>(fabsf(s) < INFINITY ? s - static_cast<float>(hi[e]) : 0.0f);
            }
            _Float16 * d = sx + (static_cast<int64_t>((k - k0) >> 5) * cols + 2 * r) * 32 + (k & 31);
            *reinterpret_cast<h4 *>(d) = hi;
            *reinterpret_cast<h4 *>(d + 32) = lo;
        }
        __syncthreads();
        for (; kb * kTileCols < k1; kb += p.wk) {
#pragma unroll
            for (int t = 0; t < TW; ++t) w[t] = w_next[t];
            const int next = min(kb + p.wk, n_kb - 1);
#pragma unroll
            for (int t = 0; t < TW; ++t) w_next[t] = wp[t][static_cast<int64_t>(next) * kWave];
            const _Float16 * xb = sx + static_cast<int64_t>((kb * kTileCols - k0) >> 5) * cols * 32 + g4 * 8;
            f4 part[TW][NB];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const bool first = (s & ((1 << p.group_shift) - 1)) == 0;
                const bool last = ((s + 1) & ((1 << p.group_shift) - 1)) == 0;
                h8 b[NB];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) b[nb] = *reinterpret_cast<const h8 *>(xb + (s * cols + bcol[nb]) * 32);
#pragma unroll
                for (int t = 0; t < TW; ++t) {
                    const h8 a = unpack(w[t][s]);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        if (first) part[t][nb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                        part[t][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b[nb], part[t][nb], 0, 0, 0);
                    }
                    if (last) {
                        const h4 d = *reinterpret_cast<const h4 *>(dp[t] + static_cast<int64_t>((kb * 4 + s) >> p.group_shift) * kTileRows);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[t][nb][i] = fmaf(part[t][nb][i], static_cast<float>(d[i]), acc[t][nb][i]);
                        }
                    }
                }
            }
        }
    }

    // the columns' waves add up in LDS, in order; the parts of x in the lanes c16 and c16 + 8
    if (p.wk > 1) {
        __syncthreads();
        f4 * sa = reinterpret_cast<f4 *>(lds);
#pragma unroll
        for (int t = 0; t < TW; ++t) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) sa[(wave * TW * NB + t * NB + nb) * kWave + lane] = acc[t][nb];
        }
        __syncthreads();
        if (wk != 0) return;
        for (int k = 1; k < p.wk; ++k) {
#pragma unroll
            for (int t = 0; t < TW; ++t) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) acc[t][nb] += sa[((wave + k) * TW * NB + t * NB + nb) * kWave + lane];
            }
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int r = nb * 8 + c16;
        f4 v[TW];
#pragma unroll
        for (int t = 0; t < TW; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[t][i] = acc[t][nb][i] + dpp_f<0x128>(acc[t][nb][i]);
        }
        if (c16 >= 8 || r >= p.rows) continue;
#pragma unroll
        for (int t = 0; t < (SWIGLU ? 1 : TW); ++t) {
            const int tile = tile0 + t;
            if (tile >= p.n_tiles) continue;
            const int o = tile * kTileRows + g4 * 4;
            float * y = p.y + static_cast<int64_t>(r) * p.out_dim + o;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (o + i >= p.out_dim) continue;
                float out = ldexpf(v[t][i], -s_exp[r]);
                if constexpr (SWIGLU) {
                    const float up = ldexpf(v[1][i], -s_exp[r]);
                    out = out / (1.0f + expf(-out)) * up;
                }
                y[i] = p.epilogue == kEpiAccumOp ? y[i] + out : out;
            }
        }
    }
}

// Packing: a workgroup takes a block of 16 rows x 128 columns, thread 16 r + s the 8 columns 8 s .. of row r.
__global__ __launch_bounds__(256) void pack_q4_kernel(const float * src, int out_dim, int in_dim, int group_shift, uint8_t * dst, _Float16 * scales) {
    const int n_kb = in_dim / kTileCols;
    const int64_t block = blockIdx.x;
    const int64_t tile = block / n_kb;
    const int kb = static_cast<int>(block - tile * n_kb);
    const int r = threadIdx.x >> 4, s = threadIdx.x & 15;
    const int64_t row = tile * kTileRows + r;
    float v[8];
    float mx = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = row < out_dim ? src[row * in_dim + kb * kTileCols + s * 8 + e] : 0.0f;   // rows behind the last are 0
        mx = fmaxf(mx, fabsf(v[e]));
    }
    // the largest of the group: 4, 8 or 16 neighbouring threads
    mx = fmaxf(mx, __shfl_xor(mx, 1, kWave));
    mx = fmaxf(mx, __shfl_xor(mx, 2, kWave));
    if (group_shift > 0) mx = fmaxf(mx, __shfl_xor(mx, 4, kWave));
    if (group_shift > 1) mx = fmaxf(mx, __shfl_xor(mx, 8, kWave));
    const _Float16 d = static_cast<_Float16>(mx / 7.0f);
    const float df = static_cast<float>(d);
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        // to the nearest of -8 .. 7, ties to even; an f16 scale that rounded down reaches past 7
        const float q = df > 0.0f ? fminf(fmaxf(rintf(v[e] / df), -8.0f), 7.0f) : 0.0f;
        w |= static_cast<uint32_t>(static_cast<int>(q) + 8) << (4 * (e >> 1) + 16 * (e & 1));
    }
    reinterpret_cast<uint32_t *>(dst)[((tile * n_kb + kb) * kWave + (s & 3) * 16 + r) * 4 + (s >> 2)] = w;
    const int per = 4 << group_shift;   // threads of a group
    if ((s & (per - 1)) == 0) {
        const int64_t group = ((static_cast<int64_t>(kb) * kTileCols + s * 8) >> 5) >> group_shift;
        scales[(tile * (in_dim >> (5 + group_shift)) + group) * kTileRows + r] = d;
    }
}

int group_shift_of(int32_t group) { return group == 32 ? 0 : group == 64 ? 1 : group == 128 ? 2 : -1; }

int check_q4(int32_t out_dim, int32_t in_dim, int32_t group, const char * who) {
    if (out_dim <= 0 || in_dim <= 0 || in_dim % kTileCols != 0 || out_dim > (1 << 24) || in_dim > (1 << 20)) {
        return fail(QA_ERR_INVALID, std::string(who) + ": in_dim a multiple of 128 up to 2^20, out_dim up to 2^24");
    }
    if (group_shift_of(group) < 0) return fail(QA_ERR_INVALID, std::string(who) + ": groups of 32, 64 or 128 columns");
    return QA_OK;
}

template <int NB, int TW, bool SWIGLU>
int launch_q4(Q4Params p, hipStream_t stream) {
    const int tiles = SWIGLU ? p.n_tiles : (p.n_tiles + TW - 1) / TW;      // units of a wave
    const int n_kb = p.in_dim / kTileCols;
    // waves of a workgroup: over the columns of a tile while the tiles alone do not fill the GPU
    p.wk = 1;
    while (p.wk < kQ4Waves && p.wk * 2 <= n_kb && static_cast<int64_t>(tiles) * p.wk < 4096) p.wk *= 2;
    p.wt = kQ4Waves / p.wk;
    // x in LDS: all of it, or whole rounds of the waves' blocks
    const int round = p.wk * kTileCols;
    p.chunk = std::min(p.in_dim, std::max(round, kXBytes / (4 * p.rows) / round * round));
    const size_t lds = std::max<size_t>(static_cast<size_t>(p.chunk) * p.rows * 4, p.wk > 1 ? static_cast<size_t>(kQ4Threads) * TW * NB * 16 : 0);
    const void * fn = reinterpret_cast<const void *>(gemv_q4_kernel<NB, TW, SWIGLU>);
    QA_HIP(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
    hipLaunchKernelGGL((gemv_q4_kernel<NB, TW, SWIGLU>), dim3(static_cast<unsigned>((tiles + p.wt - 1) / p.wt)), dim3(kQ4Threads), lds, stream, p);
    QA_LAUNCH_CHECK("gemv_q4_kernel");
    return QA_OK;
}

template <int TW, bool SWIGLU>
int launch_q4_rows(const Q4Params & p, hipStream_t stream) {
    if (p.rows <= 8) return launch_q4<1, TW, SWIGLU>(p, stream);
    if (p.rows <= 16) return launch_q4<2, TW, SWIGLU>(p, stream);
    return launch_q4<4, TW, SWIGLU>(p, stream);
}

}  // namespace
}  // namespace qa

extern "C" size_t qa_q4_weight_bytes(int32_t out_dim, int32_t in_dim) {
    using namespace qa;
    if (check_q4(out_dim, in_dim, 32, "qa_q4_weight_bytes") != QA_OK) return 0;
    return static_cast<size_t>((out_dim + kTileRows - 1) / kTileRows) * kTileRows * in_dim / 2;
}

extern "C" size_t qa_q4_scale_count(int32_t out_dim, int32_t in_dim, int32_t group) {
    using namespace qa;
    if (check_q4(out_dim, in_dim, group, "qa_q4_scale_count") != QA_OK) return 0;
    return static_cast<size_t>((out_dim + kTileRows - 1) / kTileRows) * kTileRows * (in_dim / group);
}

extern "C" int qa_pack_q4(const float * src, int32_t out_dim, int32_t in_dim, int32_t group, uint8_t * W_q4, uint16_t * scales, void * stream) {
    using namespace qa;
    if (check_q4(out_dim, in_dim, group, "qa_pack_q4") != QA_OK) return QA_ERR_INVALID;
    if (!src || !W_q4 || !scales) return fail(QA_ERR_INVALID, "qa_pack_q4: null pointer");
    if ((reinterpret_cast<uintptr_t>(W_q4) & 15) != 0 || (reinterpret_cast<uintptr_t>(scales) & 7) != 0) {
        return fail(QA_ERR_INVALID, "qa_pack_q4: weights must be aligned to 16 bytes, scales to 8");
    }
    const int64_t blocks = static_cast<int64_t>((out_dim + kTileRows - 1) / kTileRows) * (in_dim / kTileCols);
    if (blocks > INT32_MAX / 256) return fail(QA_ERR_INVALID, "qa_pack_q4: matrix too large for one call");
    if (const int rc = check_stream(stream, "qa_pack_q4"); rc != QA_OK) return rc;
    hipLaunchKernelGGL(pack_q4_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, as_stream(stream), src, out_dim, in_dim, group_shift_of(group),
                       W_q4, reinterpret_cast<_Float16 *>(scales));
    QA_LAUNCH_CHECK("pack_q4_kernel");
    return QA_OK;
}

extern "C" int qa_gemv_q4(const uint8_t * W_q4, const uint16_t * scales, int32_t group, int32_t out_dim, int32_t in_dim, const float * x,
                          int32_t rows, float * y, int32_t epilogue, const float * norm_w, float eps, void * stream) {
    using namespace qa;
    if (check_q4(out_dim, in_dim, group, "qa_gemv_q4") != QA_OK) return QA_ERR_INVALID;
    if (rows < 1 || rows > kQ4MaxRows) return fail(QA_ERR_INVALID, "qa_gemv_q4: 1 to 32 rows");
    if (epilogue < 0 || epilogue > 2) return fail(QA_ERR_INVALID, "qa_gemv_q4: epilogue 0, 1 or 2");
    if (epilogue == kEpiSwigluOp && out_dim % kTileRows != 0) return fail(QA_ERR_INVALID, "qa_gemv_q4: SwiGLU needs out_dim a multiple of 16");
    if (!W_q4 || !scales || !x || !y) return fail(QA_ERR_INVALID, "qa_gemv_q4: null pointer");
    if (((reinterpret_cast<uintptr_t>(W_q4) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(norm_w)) & 15) != 0 ||
        (reinterpret_cast<uintptr_t>(scales) & 7) != 0) {
        return fail(QA_ERR_INVALID, "qa_gemv_q4: W, x and norm_w must be aligned to 16 bytes, scales to 8");
    }
    if (const int rc = check_stream(stream, "qa_gemv_q4"); rc != QA_OK) return rc;
    Q4Params p{};
    p.W = W_q4;
    p.scales = reinterpret_cast<const _Float16 *>(scales);
    p.x = x;
    p.y = y;
    p.norm_w = norm_w;
    p.out_dim = out_dim;
    p.in_dim = in_dim;
    p.rows = rows;
    p.group_shift = group_shift_of(group);
    p.n_tiles = (out_dim + kTileRows - 1) / kTileRows;
    p.tile_up = p.n_tiles;
    p.epilogue = epilogue;
    p.eps = eps;
    if (epilogue == kEpiSwigluOp) return launch_q4_rows<2, true>(p, as_stream(stream));
    return launch_q4_rows<2, false>(p, as_stream(stream));
}
