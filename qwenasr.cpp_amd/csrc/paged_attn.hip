// Causal attention of each sequence's new tokens over a K/V cache in pages.
//
//   o_t = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q_t . k_j - m_t),   j <= n_past + t on a page that exists
//
// in one pass over the keys with a running maximum m and sum (the accumulators are rescaled when m grows).  The query
// heads of a KV head and the tokens of a sequence are columns of the same products: column c of a tile is token c / group
// and head c % group, so one token of 2 heads and a chunk of a thousand run the same code.
//
// f16 pages on v_mfma_f32_16x16x32_f16: q and p are f32, split into two f16 parts each (a power of two per column brings
// the largest |q| to 2^14..2^15, p is scaled by 2^6, so the second part keeps its bits); K and V are exact f16.  What the
// parts leave out is 2^-22 of a value, the result is as near to 64 bits as f32 products are.  Up to 8 columns carry both
// parts in one 16-column product (PACK), for decode steps.  f32 pages on v_mfma_f32_16x16x4_f32, whose products are f32.
//
// Operands without LDS.  S^T = K Q^T takes K rows as they lie: lane l holds key l % 16.  Its result leaves 4 keys of a
// column in each lane, which is the B operand of O^T = V^T P^T as it stands.  For V^T a lane loads the rows of those same
// keys, dims 8 (l % 16) .. + 7: whole rows per load instruction, and all values that it needs are its own, so the
// transposition is a register permutation (f16) or nothing at all (f32: one key per lane and product).  The output dims
// of product db are then 8 r + db for r = 0..15, 8 consecutive ones in a lane over db.
//
// What is not finite.  A masked key has p = 0, and 0 V is NaN where V is not finite; two parts of a q or p may meet an
// infinity with different signs.  The wave looks at its results once, and columns that are not finite are computed again
// key by key in f32 with only the visible keys, so that NaN appears where the formula has it and nowhere else.
#include "ops.hpp"
#include "paged.hpp"
#include "paged_device.hpp"
#include "wave.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace qa {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazyLog2 = 8.0f;    // the reference maximum follows when it is behind by more than 2^8
constexpr float kShiftLog2 = 6.0f;   // p is scaled by 2^6: at most 2^14 in f16, and its second part stays normal
constexpr int kQExp = 15;            // a column's largest |q| goes to [2^14, 2^15)
constexpr int kMaxSplits = 64;       // key ranges whose results the joining kernel adds, one lane each
// (token, head) columns of a sequence up to which the kernel of few columns takes it: one 16-column product, which on
// f16 pages carries 8 columns in two parts
constexpr int few_cols(bool f16) { return f16 ? 8 : 16; }

struct AttnParams {
    const float * q;
    const void * pages;
    float * out;
    float * part_o;       // [rows * heads][n_splits][128]
    f2 * part_ml;         // [rows * heads][n_splits]: reference maximum (log2 units) and sum
    PagedSeqs seqs;
    int32_t n_heads, n_kv, group, n_pages, page_shift, layer;
    int32_t n_tiles;      // upper bound of the tiles of the sequences this launch takes
    int32_t n_splits, split_steps;
    int32_t few_max;      // sequences of at most so many columns are the few-column kernel's
    float scale;
};

__device__ inline uint32_t lo_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ inline uint32_t hi_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ inline float row_ror8(float v) { return dpp_f<0x128>(v); }   // lane c of a row of 16 gets lane c ^ 8's

// Over the lanes c, c + 16, c + 32, c + 48, in each of them: row swaps, no LDS.
__device__ inline float column_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float column_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A tile: a sequence and its columns [col0, col0 + R).
struct Tile {
    int seq, rows, row0, past, tile, n_tiles;
};

// Tile number -> sequence: every lane counts one sequence's tiles, a prefix sum over the wave finds the one that holds
// the tile.  few: the sequences of 1..few_max columns, otherwise the longer ones.
template <int R, bool FEW>
__device__ inline Tile find_tile(const AttnParams & p, int tile, int lane) {
    for (int s0 = 0; s0 < p.seqs.n_seqs; s0 += kWave) {
        const int s = s0 + lane;
        int n = 0, rows = 0, start = 0, past = 0;
        if (s < p.seqs.n_seqs) {
            start = p.seqs.row_start[s];
            past = p.seqs.n_past[s];
            rows = rows_between(start, p.seqs.row_start[s + 1], p.seqs.n_rows);
            const bool few = static_cast<int64_t>(rows) * p.group <= p.few_max;
            if (rows > 0 && few == FEW) n = FEW ? 1 : static_cast<int>((static_cast<int64_t>(rows) * p.group + R - 1) / R);
        }
        int sum = n;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const int o = __shfl_up(sum, d, kWave);
            if (lane >= d) sum += o;
        }
        const uint64_t past_it = __ballot(sum > tile);
        if (past_it != 0) {
            const int l = __ffsll(static_cast<unsigned long long>(past_it)) - 1;
            Tile t;
            t.seq = __builtin_amdgcn_readfirstlane(s0 + l);
            t.n_tiles = __builtin_amdgcn_readlane(n, l);
            t.tile = tile - (__builtin_amdgcn_readlane(sum, l) - t.n_tiles);
            t.rows = __builtin_amdgcn_readlane(rows, l);
            t.row0 = __builtin_amdgcn_readlane(start, l);
            t.past = bounded_past(__builtin_amdgcn_readlane(past, l));
            return t;
        }
        tile -= __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    return Tile{-1, 0, 0, 0, 0, 0};
}

// Whether any position up to lim lies on a page.
__device__ inline bool sees_any(const AttnParams & p, const int32_t * table, int lim) {
    for (int j = 0; j <= lim; j += 1 << p.page_shift) {
        if (page_of(table, p.seqs.table_stride, p.page_shift, p.n_pages, j) >= 0) return true;
    }
    return false;
}

// 1 / sum, 0 for a row that sees no key; a row whose visible scores are all -inf has sum 0 and is NaN by the formula.
__device__ inline float inverse_sum(const AttnParams & p, const int32_t * table, int lim, float l) {
    if (l == 0.0f) return sees_any(p, table, lim) ? NAN : 0.0f;
    return 1.0f / l;
}

template <typename CT>
__device__ inline const CT * page_rows(const AttnParams & p, int kv, int page, int head) {
    return static_cast<const CT *>(p.pages) + cache_row_offset(p.layer, kv, page, head, 0, p.n_pages, p.n_kv, 1 << p.page_shift);
}

// One column over the visible keys of steps step0, step0 + step_inc, .. < step1, in f32, key by key: lane holds dims
// 2 lane and 2 lane + 1.  m in log2 units.
template <typename CT, int KS>
__device__ inline void column_by_keys(const AttnParams & p, const int32_t * table, int head, const float * q, int lim, int step0,
                                      int step1, int step_inc, int lane, float & m, float & l, f2 & o) {
    const f2 qv = *reinterpret_cast<const f2 *>(q + 2 * lane);
    const float c = p.scale * kLog2e;
    m = -INFINITY;
    l = 0.0f;
    o = f2{0.0f, 0.0f};
    for (int st = step0; st < step1; st += step_inc) {
        for (int j = st * KS; j < st * KS + KS && j <= lim; ++j) {
            const int page = page_of(table, p.seqs.table_stride, p.page_shift, p.n_pages, j);
            if (page < 0) continue;
            const int64_t at = static_cast<int64_t>(j & ((1 << p.page_shift) - 1)) * kHeadDim + 2 * lane;
            const CT * k = page_rows<CT>(p, 0, page, head) + at;
            const CT * v = page_rows<CT>(p, 1, page, head) + at;
            const float s = wave_sum_all(fmaf(qv[0], static_cast<float>(k[0]), qv[1] * static_cast<float>(k[1]))) * c;
            const float mn = fmaxf(m, s);
            const float ref = mn == -INFINITY ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(s - ref);
            l = l * f + e;
            o[0] = o[0] * f + e * static_cast<float>(v[0]);
            o[1] = o[1] * f + e * static_cast<float>(v[1]);
            m = mn;
        }
    }
}

// A step's K and V in registers, and whether each 16-key block of it lies on a page.
template <typename CT>
struct StepRegs;
template <>
struct StepRegs<_Float16> {
    u4 k[2][4];   // [key block][32 dims]: key l % 16, dims 32 ks + 8 (l / 16) ..
    u4 v[8];      // key 16 kb + 4 (l / 16) + i at [4 kb + i], dims 8 (l % 16) ..
};
template <>
struct StepRegs<float> {
    f4 k[8];      // key l % 16, dims 16 t + 4 (l / 16) ..
    f4 v[4][2];   // key 4 (l / 16) + i, dims 8 (l % 16) ..
};

// A column's q in MFMA order (dims 32 ks + 8 (l / 16) .. at [2 ks]); columns that do not exist are zeros.
__device__ inline void load_q(const float * qp, bool ok, int g4, f4 (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = *reinterpret_cast<const f4 *>(qp + (i >> 1) * 32 + g4 * 8 + (i & 1) * 4);
        if (!ok) x[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// Its two f16 parts, c = the score unit in log2 (scale log2 e over the column's power of two).
__device__ inline void split_q(const f4 (&x)[8], float scale, float & c, h8 (&qh)[4], h8 (&ql)[4]) {
    float mx = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(x[i][e]));
    }
    mx = column_max(mx);
    // 2^127 at most, so that it is a float; the parts of smaller q need no more
    const int ex = mx > 0.0f && mx < INFINITY ? min(kQExp - __builtin_amdgcn_frexp_expf(mx), 127) : 0;
    const float unit = ldexpf(1.0f, ex);
    c = ldexpf(scale * kLog2e, -ex);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = x[2 * ks + (e >> 2)][e & 3] * unit;        // exact: the parts add up
            qh[ks][e] = static_cast<_Float16>(v);
            ql[ks][e] = static_cast<_Float16>(v - static_cast<float>(qh[ks][e]));
        }
    }
}

// One step's scores into the running maximum, sum and probabilities; the accumulators follow a maximum that has grown.
// A masked score is -inf.
template <int NB, int KB>
__device__ inline void softmax_step(const f4 (&S)[NB][KB], const float (&c)[NB], float (&m)[NB], float (&l)[NB], f4 (&O)[NB][8],
                                    float (&pr)[NB][KB][4]) {
    float mn[NB];
    bool up[NB], any = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        float t = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) t = fmaxf(t, S[nb][kb][i]);
        }
        mn[nb] = fmaxf(m[nb], column_max(t));
        up[nb] = (mn[nb] - m[nb]) * c[nb] > kLazyLog2;   // -inf to finite: yes; -inf to -inf: NaN, no
        any = any || up[nb];
    }
    if (__any(any)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float f = up[nb] ? __builtin_amdgcn_exp2f((m[nb] - mn[nb]) * c[nb]) : 1.0f;
#pragma unroll
            for (int db = 0; db < 8; ++db) O[nb][db] *= f;
            l[nb] *= f;
            if (up[nb]) m[nb] = mn[nb];
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const float mc = m[nb] == -INFINITY ? INFINITY : fmaf(m[nb], c[nb], -kShiftLog2);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                pr[nb][kb][i] = __builtin_amdgcn_exp2f(fmaf(S[nb][kb][i], c[nb], -mc));
                l[nb] += pr[nb][kb][i];
            }
        }
    }
}

// Probabilities as two f16 parts in the order of the PV product.
__device__ inline void split_p(const float (&pr)[2][4], h8 & hi, h8 & lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float v = pr[e >> 2][e & 3];
        hi[e] = static_cast<_Float16>(v);
        lo[e] = static_cast<_Float16>(v - static_cast<float>(hi[e]));
    }
}

// 4 values of a column from dim on: the output, or the part of this split (lead: this lane also stores the part's weights).
__device__ inline void store_column(const AttnParams & p, const int32_t * table, int split, int row, int lim, int dim, f4 v, float mc,
                                    float l, bool lead) {
    if (p.n_splits == 1) {
        *reinterpret_cast<f4 *>(p.out + static_cast<int64_t>(row) * kHeadDim + dim) = v * inverse_sum(p, table, lim, l);
    } else {
        const int64_t at = static_cast<int64_t>(row) * p.n_splits + split;
        *reinterpret_cast<f4 *>(p.part_o + at * kHeadDim + dim) = v;
        if (lead) p.part_ml[at] = f2{mc, l};
    }
}

// The end of a wave's steps: the column's sum over its 4 lanes, its reference in log2 units, and the columns of each block
// whose values are not all finite.
template <int NB, bool PACK>
__device__ inline void close_columns(const int (&orow)[NB], const float (&c)[NB], const float (&m)[NB], float (&l)[NB], f4 (&O)[NB][8],
                                     float (&mc)[NB], uint32_t (&redo)[NB]) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        l[nb] = column_sum(l[nb]);
        mc[nb] = m[nb] == -INFINITY ? -INFINITY : fmaf(m[nb], c[nb], -kShiftLog2);
        // 0 x is 0 unless x is not finite, and a sum of such products is then NaN
        float zero = 0.0f * l[nb];
#pragma unroll
        for (int db = 0; db < 8; ++db) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (PACK) O[nb][db][i] += row_ror8(O[nb][db][i]);
                zero = fmaf(0.0f, O[nb][db][i], zero);
            }
        }
        const uint64_t bad = __ballot((!(zero == 0.0f) || m[nb] == INFINITY) && orow[nb] >= 0);
        redo[nb] = static_cast<uint32_t>(bad | (bad >> 16) | (bad >> 32) | (bad >> 48)) & (PACK ? 0xffu : 0xffffu);
    }
}

// The flagged columns of a block, key by key; their values are stored at once.
template <typename CT, int KS>
__device__ inline void redo_columns(const AttnParams & p, const int32_t * table, int head, int split, int lane, int lim, int orow,
                                    uint32_t redo, int step_lo, int step_hi) {
    for (uint32_t left = redo; left != 0; left &= left - 1) {
        const int col = __ffs(left) - 1;
        const int row = __builtin_amdgcn_readlane(orow, col), lm = __builtin_amdgcn_readlane(lim, col);
        float cm, cl;
        f2 co;
        column_by_keys<CT, KS>(p, table, head, p.q + static_cast<int64_t>(row) * kHeadDim, lm, step_lo, step_hi, 1, lane, cm, cl, co);
        const f2 nx = f2{__shfl_down(co[0], 1, kWave), __shfl_down(co[1], 1, kWave)};
        if ((lane & 1) == 0) store_column(p, table, split, row, lm, 2 * lane, f4{co[0], co[1], nx[0], nx[1]}, cm, cl, lane == 0);
    }
}

// Stores the columns of a wave that holds all of a split's steps.
template <typename CT, int NB, int KS>
__device__ inline void store_columns(const AttnParams & p, const int32_t * table, int head, int split, int lane, const int (&lim)[NB],
                                     const int (&orow)[NB], const float (&mc)[NB], const float (&l)[NB], const f4 (&O)[NB][8],
                                     const uint32_t (&redo)[NB], int step_lo, int step_hi) {
    const int c16 = lane & 15, g4 = lane >> 4;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        if (orow[nb] >= 0 && !((redo[nb] >> c16) & 1)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f4 a, b;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    a[e] = O[nb][e][i];
                    b[e] = O[nb][4 + e][i];
                }
                store_column(p, table, split, orow[nb], lim[nb], (g4 * 4 + i) * 8, a, mc[nb], l[nb], i == 0 && g4 == 0);
                store_column(p, table, split, orow[nb], lim[nb], (g4 * 4 + i) * 8 + 4, b, mc[nb], l[nb], false);
            }
        }
        redo_columns<CT, KS>(p, table, head, split, lane, lim[nb], orow[nb], redo[nb], step_lo, step_hi);
    }
}

// The kernel.  NB blocks of 16 columns per wave, WC waves side by side over columns, WK waves over the steps of the keys
// (merged in LDS).  A step is 32 keys of f16 or 16 keys of f32: 8 KB of K and 8 KB of V either way.
template <typename CT, int NB, int WC, int WK, bool FEW>
__global__ __launch_bounds__(kWave * WC * WK, NB == 1 ? 3 : 2) void paged_attn_kernel(AttnParams p) {
    constexpr bool F16 = std::is_same<CT, _Float16>::value;
    constexpr bool PACK = FEW && F16;                // one block of 8 columns in two parts
    static_assert(!FEW || (NB == 1 && WC == 1), "the kernel of few columns has one block of them");
    constexpr int KS = F16 ? 32 : 16, KB = F16 ? 2 : 1;
    constexpr int kCols = PACK ? 8 : NB * 16;        // a wave's columns
    constexpr int R = WC * kCols;                    // the tile's
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wc = wave % WC, wk = wave / WC;
    const int c16 = lane & 15, g4 = lane >> 4;

    // block -> (split, tile, KV head): neighbouring blocks, which go to different XCDs, take different heads
    const int head = static_cast<int>(blockIdx.x) % p.n_kv;
    const int rest = static_cast<int>(blockIdx.x) / p.n_kv;
    const int split = rest / p.n_tiles;
    const Tile tl = find_tile<R, FEW>(p, rest - split * p.n_tiles, lane);
    if (tl.seq < 0) return;
    const int col0 = (tl.n_tiles - 1 - tl.tile) * R;                  // the last tile has the most keys: first
    const int n_cols = tl.rows * p.group;
    const int cap = p.seqs.table_stride << p.page_shift;
    const int32_t * table = p.seqs.tables + static_cast<int64_t>(tl.seq) * p.seqs.table_stride;
    const int t_first = col0 / p.group, t_last = (min(col0 + R, n_cols) - 1) / p.group;
    const int kend = max(0, min(tl.past + t_last, cap - 1) + 1);      // keys that the tile's last token sees
    const int n_steps = (kend + KS - 1) / KS;
    const int step_lo = split * p.split_steps;
    const int step_hi = split == p.n_splits - 1 ? n_steps : min(n_steps, step_lo + p.split_steps);
    if (split > 0 && step_lo >= n_steps) return;                      // uniform for the workgroup
    const int full = max(0, min(tl.past + t_first, cap - 1) + 1) / KS;   // steps that every column sees whole

    // columns: q in MFMA order, visible keys, output row
    int lim[NB], orow[NB];
    float c[NB];
    h8 qh[F16 ? NB : 1][4], ql[F16 ? NB : 1][4];
    f4 qf[F16 ? 1 : NB][8];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int col = col0 + wc * kCols + nb * 16 + (PACK ? c16 & 7 : c16);
        const bool ok = col < n_cols;
        const int t = ok ? col / p.group : t_last;
        const int h = ok ? col - t * p.group : 0;
        lim[nb] = ok ? min(tl.past + t, cap - 1) : kend - 1;
        orow[nb] = ok ? (tl.row0 + t) * p.n_heads + head * p.group + h : -1;
        const float * qp = p.q + (static_cast<int64_t>(tl.row0 + t) * p.n_heads + head * p.group + h) * kHeadDim;
        if constexpr (F16) {
            f4 x[8];
            load_q(qp, ok, g4, x);
            split_q(x, p.scale, c[nb], qh[nb], ql[nb]);
            if constexpr (PACK) {
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) qh[nb][ks] = c16 < 8 ? qh[nb][ks] : ql[nb][ks];
            }
        } else {
            c[nb] = p.scale * kLog2e;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                qf[nb][i] = *reinterpret_cast<const f4 *>(qp + i * 16 + g4 * 4);
                if (!ok) qf[nb][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
    }

    float m[NB], l[NB];
    f4 O[NB][8];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        m[nb] = -INFINITY;
        l[nb] = 0.0f;
#pragma unroll
        for (int db = 0; db < 8; ++db) O[nb][db] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // the page of each 16-key block of a step, -1 for none (uniform)
    auto pages_of = [&](int st, int (&pg)[KB]) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const int j = st * KS + kb * 16;
            pg[kb] = j < kend ? page_of(table, p.seqs.table_stride, p.page_shift, p.n_pages, j) : -1;
        }
    };
    const int in_page = (1 << p.page_shift) - 1;
    StepRegs<CT> r;
    auto load_k = [&](int st, const int (&pg)[KB]) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            // a block on no page reads page 0, which there always is, and is masked
            const CT * base = page_rows<CT>(p, 0, max(pg[kb], 0), head) + static_cast<int64_t>((st * KS + kb * 16) & in_page) * kHeadDim;
            if constexpr (F16) {
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) r.k[kb][ks] = *reinterpret_cast<const u4 *>(base + c16 * kHeadDim + ks * 32 + g4 * 8);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) r.k[i] = *reinterpret_cast<const f4 *>(base + c16 * kHeadDim + i * 16 + g4 * 4);
            }
        }
    };
    auto load_v = [&](int st, const int (&pg)[KB]) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const CT * base = page_rows<CT>(p, 1, max(pg[kb], 0), head) + static_cast<int64_t>((st * KS + kb * 16) & in_page) * kHeadDim;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const CT * v = base + (g4 * 4 + i) * kHeadDim + c16 * 8;
                if constexpr (F16) {
                    r.v[kb * 4 + i] = *reinterpret_cast<const u4 *>(v);
                } else {
                    r.v[i][0] = *reinterpret_cast<const f4 *>(v);
                    r.v[i][1] = *reinterpret_cast<const f4 *>(v + 4);
                }
            }
        }
    };

    int st = step_lo + wk;
    int pg[KB], pg_next[KB];
    if (st < step_hi) {
        pages_of(st, pg);
        load_k(st, pg);
        load_v(st, pg);
        pages_of(min(st + WK, n_steps - 1), pg_next);
    }
    for (; st < step_hi; st += WK) {
        const bool more = st + WK < step_hi;
        bool hole = false;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) hole = hole || pg[kb] < 0;

        f4 S[NB][KB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                S[nb][kb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        if constexpr (F16) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const h8 a = __builtin_bit_cast(h8, r.k[kb][ks]);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        S[nb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[nb][ks], S[nb][kb], 0, 0, 0);
                        if constexpr (!PACK) S[nb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[nb][ks], S[nb][kb], 0, 0, 0);
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) S[nb][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(r.k[i][e], qf[nb][i][e], S[nb][0], 0, 0, 0);
                }
            }
        }
        if (more) load_k(st + WK, pg_next);
        if constexpr (PACK) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
                for (int i = 0; i < 4; ++i) S[0][kb][i] += row_ror8(S[0][kb][i]);
            }
        }
        if (st >= full || hole) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (st * KS + kb * 16 + g4 * 4 + i > lim[nb] || pg[kb] < 0) S[nb][kb][i] = -INFINITY;
                    }
                }
            }
        }

        float pr[NB][KB][4];
        softmax_step<NB, KB>(S, c, m, l, O, pr);

        // rows of keys that no column sees, and of no page, are whatever memory holds: not even 0 times that
        if (st * KS + KS > kend || hole) {
            if constexpr (F16) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (st * KS + (e >> 2) * 16 + g4 * 4 + (e & 3) >= kend || pg[e >> 2] < 0) r.v[e] = u4{0, 0, 0, 0};
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (st * KS + g4 * 4 + i >= kend || pg[0] < 0) r.v[i][0] = r.v[i][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
        }
        if constexpr (F16) {
            h8 ph[NB], pl[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                split_p(pr[nb], ph[nb], pl[nb]);
                if constexpr (PACK) ph[nb] = c16 < 8 ? ph[nb] : pl[nb];
            }
#pragma unroll
            for (int db = 0; db < 8; ++db) {
                u4 a;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t x = r.v[2 * w][db >> 1], y = r.v[2 * w + 1][db >> 1];
                    a[w] = db & 1 ? hi_pair(x, y) : lo_pair(x, y);
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    O[nb][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), ph[nb], O[nb][db], 0, 0, 0);
                    if constexpr (!PACK) O[nb][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), pl[nb], O[nb][db], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int db = 0; db < 8; ++db) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        O[nb][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(r.v[i][db >> 2][db & 3], pr[nb][0][i], O[nb][db], 0, 0, 0);
                    }
                }
            }
        }
        if (more) {
            load_v(st + WK, pg_next);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) pg[kb] = pg_next[kb];
            pages_of(min(st + 2 * WK, n_steps - 1), pg_next);
        }
    }

    float mc[NB];
    uint32_t redo[NB];
    close_columns<NB, PACK>(orow, c, m, l, O, mc, redo);
    if constexpr (WK == 1) {
        store_columns<CT, NB, KS>(p, table, head, split, lane, lim, orow, mc, l, O, redo, step_lo, step_hi);
    } else {
        // merge over the WK waves of a column in LDS
        constexpr int kStride = kHeadDim + 4;
        __shared__ __attribute__((aligned(16))) float so[WK * R * kStride];
        __shared__ float sm[WK * R], sl[WK * R];
        __shared__ int srow[R], slim[R];
        const int base = wk * R + wc * kCols;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            if (!PACK || c16 < 8) {
                const int at = base + nb * 16 + c16;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    f4 a, b;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[e] = O[nb][e][i];
                        b[e] = O[nb][4 + e][i];
                    }
                    *reinterpret_cast<f4 *>(so + at * kStride + (g4 * 4 + i) * 8) = a;
                    *reinterpret_cast<f4 *>(so + at * kStride + (g4 * 4 + i) * 8 + 4) = b;
                }
                if (g4 == 0) {
                    sm[at] = mc[nb];
                    sl[at] = l[nb];
                    if (wk == 0) {
                        srow[wc * kCols + nb * 16 + c16] = orow[nb];
                        slim[wc * kCols + nb * 16 + c16] = lim[nb];
                    }
                }
            }
            for (uint32_t left = redo[nb]; left != 0; left &= left - 1) {
                const int col = __ffs(left) - 1;
                const int row = __builtin_amdgcn_readlane(orow[nb], col), lm = __builtin_amdgcn_readlane(lim[nb], col);
                float cm, cl;
                f2 co;
                column_by_keys<CT, KS>(p, table, head, p.q + static_cast<int64_t>(row) * kHeadDim, lm, step_lo + wk, step_hi, WK, lane,
                                       cm, cl, co);
                // after this wave's own stores above: one wave's LDS accesses stay in order
                __builtin_amdgcn_wave_barrier();
                const int at = base + nb * 16 + col;
                *reinterpret_cast<f2 *>(so + at * kStride + 2 * lane) = co;
                if (lane == 0) {
                    sm[at] = cm;
                    sl[at] = cl;
                }
            }
        }
        __syncthreads();
        for (int idx = threadIdx.x; idx < R * (kHeadDim / 4); idx += kWave * WC * WK) {
            const int col = idx / (kHeadDim / 4), dim = (idx % (kHeadDim / 4)) * 4;
            const int row = srow[col];
            if (row < 0) continue;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < WK; ++w) M = fmaxf(M, sm[w * R + col]);
            float ls = 0.0f;
            f4 o = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                const float mw = sm[w * R + col];
                const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - M);
                ls += sl[w * R + col] * f;
                o += *reinterpret_cast<const f4 *>(so + (w * R + col) * kStride + dim) * f;
            }
            store_column(p, table, split, row, slim[col], dim, o, M, ls, dim == 0);
        }
    }
}

// The kernel of long chunks on f16 pages: 4 waves of 32 columns each share the K and V of a tile through LDS, which cuts
// what the CUs pull from L2 to a quarter (without it that traffic sets the pace).  A tile is 64 keys, two steps of 32; a
// step lies in LDS as the MFMA operands themselves, 8 of K and 8 of V^T, 64 lanes x 16 bytes each: every read and write is
// one unbroken kilobyte and no wave rearranges anything.  Waves 0 and 1 fetch and transpose V of the two steps, waves 2 and
// 3 fetch K.  Two tiles in LDS, the next one's rows in registers: one barrier per tile, and two workgroups per CU, each
// multiplying while the other waits at its barrier.
constexpr int kTileSteps = 2;
constexpr int kTileWaves = 2 * kTileSteps, kTileColumns = kTileWaves * 32;
constexpr int kStepHalfs = 16 * kWave * 8;   // a step's 16 operands
constexpr size_t kTileLds = 2 * kTileSteps * kStepHalfs * sizeof(_Float16);
constexpr int kOutStride = kHeadDim + 4, kOutFloats = 16 * kOutStride;   // a wave's 16 columns on their way out
static_assert(kTileWaves * kOutFloats * sizeof(float) <= kTileLds, "the outputs go through the operands' LDS");

__global__ __launch_bounds__(kTileWaves * kWave, 2) void paged_attn_tile_kernel(AttnParams p) {
    constexpr int NB = 2;
    extern __shared__ __attribute__((aligned(16))) _Float16 lds_kv[];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    const int head = static_cast<int>(blockIdx.x) % p.n_kv;
    const int rest = static_cast<int>(blockIdx.x) / p.n_kv;
    const int split = rest / p.n_tiles;
    const Tile tl = find_tile<kTileColumns, false>(p, rest - split * p.n_tiles, lane);
    if (tl.seq < 0) return;
    const int col0 = (tl.n_tiles - 1 - tl.tile) * kTileColumns;
    const int n_cols = tl.rows * p.group;
    const int cap = p.seqs.table_stride << p.page_shift;
    const int32_t * table = p.seqs.tables + static_cast<int64_t>(tl.seq) * p.seqs.table_stride;
    const int t_last = (min(col0 + kTileColumns, n_cols) - 1) / p.group;
    const int kend = max(0, min(tl.past + t_last, cap - 1) + 1);
    const int n_steps = (kend + 31) / 32;
    const int step_lo = split * p.split_steps;
    const int step_hi = split == p.n_splits - 1 ? n_steps : min(n_steps, step_lo + p.split_steps);
    if (split > 0 && step_lo >= n_steps) return;                      // uniform for the workgroup
    const int in_page = (1 << p.page_shift) - 1;

    // columns: their q is on its way while the first tile is fetched
    int lim[NB], orow[NB];
    f4 x[NB][8];
    int wave_lim = -1, wave_first = 1 << 30;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int col = col0 + wave * 32 + nb * 16 + c16;
        const bool ok = col < n_cols;
        const int t = ok ? col / p.group : t_last;
        const int h = ok ? col - t * p.group : 0;
        lim[nb] = ok ? min(tl.past + t, cap - 1) : -1;
        orow[nb] = ok ? (tl.row0 + t) * p.n_heads + head * p.group + h : -1;
        load_q(p.q + (static_cast<int64_t>(tl.row0 + t) * p.n_heads + head * p.group + h) * kHeadDim, ok, g4, x[nb]);
    }
    {
        // keys that the wave's last and first token see (its columns are in order of token)
        const int first_col = col0 + wave * 32, last_col = min(first_col + 32, n_cols) - 1;
        if (first_col < n_cols) {
            wave_first = min(tl.past + first_col / p.group, cap - 1);
            wave_lim = min(tl.past + last_col / p.group, cap - 1);
        }
    }
    const int wave_steps = min(step_hi, (wave_lim + 32) / 32);        // steps behind it hold nothing that the wave sees
    const int full = max(0, wave_first + 1) / 32;

    // this wave's share of a tile: step `wave % 4`, V (waves 0..3) or K
    const bool fetch_v = wave < kTileSteps;
    u4 r[8];
    int pg[2];
    __shared__ int s_holes[2][kTileSteps];                            // bit kb: 16-key block kb of the step lies on no page
    // table entries of a step's two 16-key blocks as they are, looked at when they have arrived
    auto entries_of = [&](int st, int (&out)[2]) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) out[kb] = table[min((st * 32 + kb * 16) >> p.page_shift, p.seqs.table_stride - 1)];
    };
    int st_held = 0;
    auto fetch = [&](int st, const int (&from)[2]) {
        st_held = st;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            pg[kb] = st * 32 + kb * 16 < kend && from[kb] >= 0 && from[kb] < p.n_pages ? from[kb] : -1;
            const _Float16 * base = page_rows<_Float16>(p, fetch_v ? 1 : 0, max(pg[kb], 0), head) +
                                    static_cast<int64_t>((st * 32 + kb * 16) & in_page) * kHeadDim;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // V: row 4 g4 + i, dims 8 c16 ..; K: row c16, dims 32 i + 8 g4 ..
                const int off = fetch_v ? (g4 * 4 + i) * kHeadDim + c16 * 8 : c16 * kHeadDim + i * 32 + g4 * 8;
                r[kb * 4 + i] = *reinterpret_cast<const u4 *>(base + off);
            }
        }
    };
    auto put = [&](int buf) {
        _Float16 * to = lds_kv + (buf * kTileSteps + (wave & (kTileSteps - 1))) * kStepHalfs + lane * 8;
        if (fetch_v) {
            if (st_held * 32 + 32 > kend || pg[0] < 0 || pg[1] < 0) {   // rows that no column sees, and of no page: not even 0 times them
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (st_held * 32 + (e >> 2) * 16 + g4 * 4 + (e & 3) >= kend || pg[e >> 2] < 0) r[e] = u4{0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int db = 0; db < 8; ++db) {
                u4 a;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    a[w] = db & 1 ? hi_pair(r[2 * w][db >> 1], r[2 * w + 1][db >> 1]) : lo_pair(r[2 * w][db >> 1], r[2 * w + 1][db >> 1]);
                }
                *reinterpret_cast<u4 *>(to + (8 + db) * kWave * 8) = a;
            }
        } else {
#pragma unroll
            for (int f = 0; f < 8; ++f) *reinterpret_cast<u4 *>(to + f * kWave * 8) = r[f];
            if (lane == 0) s_holes[buf][wave & (kTileSteps - 1)] = (pg[0] < 0 ? 1 : 0) | (pg[1] < 0 ? 2 : 0);
        }
    };

    const int mine = wave & (kTileSteps - 1);
    const int n_tiles = (step_hi - step_lo + kTileSteps - 1) / kTileSteps;
    int pg_next[2];
    if (n_tiles > 0) {
        entries_of(step_lo + mine, pg_next);
        fetch(step_lo + mine, pg_next);
        entries_of(step_lo + kTileSteps + mine, pg_next);
    }

    float c[NB];
    h8 qh[NB][4], ql[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) split_q(x[nb], p.scale, c[nb], qh[nb], ql[nb]);
    float m[NB], l[NB];
    f4 O[NB][8];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        m[nb] = -INFINITY;
        l[nb] = 0.0f;
#pragma unroll
        for (int db = 0; db < 8; ++db) O[nb][db] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (n_tiles > 0) {
        put(0);
        fetch(step_lo + kTileSteps + mine, pg_next);
        entries_of(step_lo + 2 * kTileSteps + mine, pg_next);
    }
    __syncthreads();
    for (int tile = 0; tile < n_tiles; ++tile) {
        const _Float16 * buf = lds_kv + (tile & 1) * kTileSteps * kStepHalfs + lane * 8;
        const int st0 = step_lo + tile * kTileSteps;
#pragma unroll 1
        for (int s = 0; s < kTileSteps; ++s) {
            const int st = st0 + s;
            if (st >= wave_steps) break;                              // uniform for the wave
            const _Float16 * op = buf + s * kStepHalfs;
            f4 S[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) S[nb][0] = S[nb][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            h8 a[8];
#pragma unroll
            for (int f = 0; f < 8; ++f) a[f] = *reinterpret_cast<const h8 *>(op + f * kWave * 8);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) S[nb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[kb * 4 + ks], qh[nb][ks], S[nb][kb], 0, 0, 0);
                }
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) S[nb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[kb * 4 + ks], ql[nb][ks], S[nb][kb], 0, 0, 0);
                }
            }
            h8 v[8];
#pragma unroll
            for (int db = 0; db < 8; ++db) v[db] = *reinterpret_cast<const h8 *>(op + (8 + db) * kWave * 8);
            const int holes = __builtin_amdgcn_readfirstlane(s_holes[tile & 1][s]);
            if (st >= full || holes != 0) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (st * 32 + kb * 16 + g4 * 4 + i > lim[nb] || ((holes >> kb) & 1)) S[nb][kb][i] = -INFINITY;
                        }
                    }
                }
            }
            float pr[NB][2][4];
            softmax_step<NB, 2>(S, c, m, l, O, pr);
            h8 ph[NB], pl[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) split_p(pr[nb], ph[nb], pl[nb]);
#pragma unroll
            for (int db = 0; db < 8; ++db) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) O[nb][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[db], ph[nb], O[nb][db], 0, 0, 0);
            }
#pragma unroll
            for (int db = 0; db < 8; ++db) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) O[nb][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[db], pl[nb], O[nb][db], 0, 0, 0);
            }
        }
        if (tile + 1 < n_tiles) {
            put((tile + 1) & 1);
            if (tile + 2 < n_tiles) {
                fetch(st0 + 2 * kTileSteps + mine, pg_next);
                entries_of(st0 + 3 * kTileSteps + mine, pg_next);
            }
        }
        __syncthreads();
    }
    float mc[NB];
    uint32_t redo[NB];
    close_columns<NB, false>(orow, c, m, l, O, mc, redo);
    // through the wave's own part of LDS, so that a store instruction writes two whole rows; a lane's values would lie 16 bytes
    // in each of 64 lines
    float * so = reinterpret_cast<float *>(lds_kv) + wave * kOutFloats;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        float * to = so + c16 * kOutStride + g4 * 32;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                *reinterpret_cast<f4 *>(to + i * 8 + h * 4) = f4{O[nb][4 * h][i], O[nb][4 * h + 1][i], O[nb][4 * h + 2][i], O[nb][4 * h + 3][i]};
            }
        }
        // lane -> column 2 i + lane / 32, dims 4 (lane % 32) ..; what belongs to a column comes from its lane
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int col = 2 * i + (lane >> 5), dim = (lane & 31) * 4;
            const int row = __shfl(orow[nb], col, kWave), lm = __shfl(lim[nb], col, kWave);
            const float cm = __shfl(mc[nb], col, kWave), cl = __shfl(l[nb], col, kWave);
            const f4 v = *reinterpret_cast<const f4 *>(so + col * kOutStride + dim);
            if (row >= 0 && !((redo[nb] >> col) & 1)) store_column(p, table, split, row, lm, dim, v, cm, cl, dim == 0);
        }
        redo_columns<_Float16, 32>(p, table, head, split, lane, lim[nb], orow[nb], redo[nb], step_lo, step_hi);
    }
}

// Joins the splits of each (row, head): one wave each, lane = split for the weights, then lane = 2 dims.  Its time is
// dependent loads, so the sequences, the weights and the first results are read together; a split that the row does not
// reach holds whatever the workspace held, and is selected away.
__global__ __launch_bounds__(256) void paged_join_kernel(AttnParams p, int ks) {
    constexpr int kFirst = 8;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= static_cast<int64_t>(p.seqs.n_rows) * p.n_heads) return;
    const int row = static_cast<int>(item / p.n_heads);
    const float * po = p.part_o + item * p.n_splits * kHeadDim + 2 * lane;
    f2 ml = p.part_ml[item * p.n_splits + min(lane, p.n_splits - 1)];
    f2 part[kFirst];
#pragma unroll
    for (int s = 0; s < kFirst; ++s) part[s] = *reinterpret_cast<const f2 *>(po + min(s, p.n_splits - 1) * kHeadDim);
    const RowPlace at = row_place(p.seqs, row, lane);
    if (at.seq < 0) return;
    const int cap = p.seqs.table_stride << p.page_shift;
    const int lim = min(at.pos, cap - 1);
    // splits that hold a key which this row sees (the first is always computed)
    const int active = lim < 0 ? 1 : min(p.n_splits, lim / ks / p.split_steps + 1);
    if (lane >= active) ml = f2{-INFINITY, 0.0f};
    const float M = wave_max_all(ml[0]);
    const float f = ml[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[0] - M);
    const float L = wave_sum_all(ml[1] * f);
    f2 o = f2{0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < kFirst; ++s) {
        const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), s));
        if (s < active) o += part[s] * w;
    }
    for (int s0 = kFirst; s0 < active; s0 += kFirst) {
#pragma unroll
        for (int s = 0; s < kFirst; ++s) part[s] = *reinterpret_cast<const f2 *>(po + min(s0 + s, active - 1) * kHeadDim);
#pragma unroll
        for (int s = 0; s < kFirst; ++s) {
            if (s0 + s < active) o += part[s] * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), s0 + s));
        }
    }
    const float inv = inverse_sum(p, p.seqs.tables + static_cast<int64_t>(at.seq) * p.seqs.table_stride, lim, L);
    *reinterpret_cast<f2 *>(p.out + item * kHeadDim + 2 * lane) = o * inv;
}

constexpr int kMidCols = 64;   // columns of a sequence up to which waves share no LDS tile

// How a call cuts its work: which kernels run, their upper bounds of tiles, and the key ranges.
struct AttnPlan {
    bool few;                // sequences of few columns, when the host's bounds allow any
    int many_cols;           // columns of a tile of the other kernel, 0: all sequences are of few
    int tiles_few, tiles_many;
    int splits, split_steps; // of both, in steps of the cache type
};

AttnPlan attn_plan(const qa_kv_layout & l, const qa_paged_batch & b, int32_t n_heads, size_t workspace_bytes) {
    const bool f16 = l.cache_type == QA_CACHE_F16;
    const int ks = f16 ? 32 : 16;
    const int group = n_heads / l.n_kv_heads;
    const int seqs = std::min(b.n_seqs, b.n_rows);
    const int64_t most = std::min<int64_t>(b.n_rows, b.max_tokens > 0 ? b.max_tokens : b.n_rows);
    const int64_t cols = static_cast<int64_t>(b.n_rows) * group;
    AttnPlan pl{};
    // one sequence is either; the host's bounds say whether all are of few columns
    if (most * group > few_cols(f16)) pl.many_cols = f16 ? (most * group > kMidCols ? kTileColumns : 64) : 64;
    pl.few = pl.many_cols == 0 || b.n_seqs > 1;
    pl.tiles_few = seqs;
    pl.tiles_many = pl.many_cols ? static_cast<int>(cols / pl.many_cols + seqs) : 0;
    const int64_t cap = static_cast<int64_t>(b.table_stride) * l.max_seq;
    const int64_t len = std::min<int64_t>(cap, b.max_len > 0 ? b.max_len : cap);
    const int steps = static_cast<int>((len + ks - 1) / ks);
    const int64_t tiles = pl.many_cols ? std::max<int64_t>(1, (cols + pl.many_cols - 1) / pl.many_cols) : pl.tiles_few;
    const int64_t target = pl.many_cols == kTileColumns ? 512 : 1024, least = pl.many_cols == kTileColumns ? 4 : 8;
    int64_t splits = std::max<int64_t>(1, std::min<int64_t>({target / std::max<int64_t>(tiles * l.n_kv_heads, 1), (steps + least - 1) / least, kMaxSplits}));
    const size_t per_split = static_cast<size_t>(b.n_rows) * n_heads * (kHeadDim + 2) * sizeof(float);
    if (splits > 1 && per_split * splits > workspace_bytes) splits = std::max<int64_t>(1, static_cast<int64_t>(workspace_bytes / per_split));
    pl.split_steps = std::max<int>(1, static_cast<int>((steps + splits - 1) / splits));
    pl.splits = std::max(1, (steps + pl.split_steps - 1) / pl.split_steps);
    return pl;
}

template <typename CT>
int launch_attn(const AttnPlan & pl, AttnParams p, hipStream_t stream) {
    constexpr bool F16 = std::is_same<CT, _Float16>::value;
    const unsigned per = static_cast<unsigned>(p.n_kv) * pl.splits;
    p.few_max = pl.few ? few_cols(F16) : 0;
    if (pl.many_cols) {
        p.n_tiles = pl.tiles_many;
        if constexpr (!F16) {
            hipLaunchKernelGGL((paged_attn_kernel<CT, 1, 4, 1, false>), dim3(per * p.n_tiles), dim3(256), 0, stream, p);
        } else if (pl.many_cols == kTileColumns) {
            QA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(paged_attn_tile_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(kTileLds)));
            hipLaunchKernelGGL(paged_attn_tile_kernel, dim3(per * p.n_tiles), dim3(kTileWaves * kWave), kTileLds, stream, p);
        } else {
            hipLaunchKernelGGL((paged_attn_kernel<CT, 2, 2, 2, false>), dim3(per * p.n_tiles), dim3(256), 0, stream, p);
        }
    }
    if (pl.few) {
        p.n_tiles = pl.tiles_few;
        hipLaunchKernelGGL((paged_attn_kernel<CT, 1, 1, 4, true>), dim3(per * p.n_tiles), dim3(256), 0, stream, p);
    }
    if (pl.splits > 1) {
        const int64_t items = static_cast<int64_t>(p.seqs.n_rows) * p.n_heads;
        hipLaunchKernelGGL(paged_join_kernel, dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256), 0, stream, p, F16 ? 32 : 16);
    }
    QA_LAUNCH_CHECK("paged_attn_kernel");
    return QA_OK;
}

}  // namespace
}  // namespace qa

extern "C" size_t qa_paged_attn_workspace_bytes(const qa_kv_layout * layout, const qa_paged_batch * batch, int32_t n_heads) {
    using namespace qa;
    if (check_batch(layout, 0, batch, n_heads, "qa_paged_attn_workspace_bytes") != QA_OK || batch->n_rows == 0) return 0;
    const AttnPlan pl = attn_plan(*layout, *batch, n_heads, SIZE_MAX);
    if (pl.splits <= 1) return 0;
    return static_cast<size_t>(batch->n_rows) * n_heads * pl.splits * (kHeadDim + 2) * sizeof(float);
}

extern "C" int qa_paged_attn(const float * q, const void * pages, const qa_kv_layout * layout, int32_t layer,
                             const qa_paged_batch * batch, int32_t n_heads, float scale, float * out, void * workspace,
                             size_t workspace_bytes, void * stream) {
    using namespace qa;
    if (check_batch(layout, layer, batch, n_heads, "qa_paged_attn") != QA_OK) return QA_ERR_INVALID;
    if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(QA_ERR_INVALID, "qa_paged_attn: scale must be positive and finite");
    if (batch->n_rows == 0) return QA_OK;
    if (!q || !pages || !out || (!workspace && workspace_bytes > 0)) return fail(QA_ERR_INVALID, "qa_paged_attn: null pointer");
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(out) |
          reinterpret_cast<uintptr_t>(workspace)) & 15) != 0) {
        return fail(QA_ERR_INVALID, "qa_paged_attn: pointers must be aligned to 16 bytes");
    }
    if (static_cast<int64_t>(batch->n_rows) * n_heads > INT32_MAX) return fail(QA_ERR_INVALID, "qa_paged_attn: too many rows");
    if (const int rc = check_stream(stream, "qa_paged_attn"); rc != QA_OK) return rc;
    const AttnPlan pl = attn_plan(*layout, *batch, n_heads, workspace_bytes);
    if (static_cast<int64_t>(std::max(pl.tiles_many, pl.tiles_few)) * layout->n_kv_heads * pl.splits > INT32_MAX / 256) {
        return fail(QA_ERR_INVALID, "qa_paged_attn: too many rows");
    }
    AttnParams p{};
    p.q = q;
    p.pages = pages;
    p.out = out;
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = reinterpret_cast<f2 *>(p.part_o + static_cast<int64_t>(batch->n_rows) * n_heads * pl.splits * kHeadDim);
    p.seqs = paged_seqs(*batch);
    p.n_heads = n_heads;
    p.n_kv = layout->n_kv_heads;
    p.group = n_heads / layout->n_kv_heads;
    p.n_pages = layout->n_streams;
    p.page_shift = page_shift_of(layout->max_seq);
    p.layer = layer;
    p.n_splits = pl.splits;
    p.split_steps = pl.split_steps;
    p.scale = scale;
    return layout->cache_type == QA_CACHE_F16 ? launch_attn<_Float16>(pl, p, as_stream(stream)) : launch_attn<float>(pl, p, as_stream(stream));
}
