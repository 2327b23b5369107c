// Matrix-vector products with 4-bit weights: y = W x for 1 to 32 token rows, w = (q - 8) d, q in 0..15, d an f16 scale per
// row and group of 32, 64 or 128 columns, with the RMSNorm before and the SwiGLU behind that the decoder's GEMVs fuse.
//
// What bounds it is the stream of W: half a byte per weight, 1/8 of the f32 GEMV's.  A block of 16 rows x 128 columns is
// 1 KB, one 16-byte load per lane, and lies in the order in which v_mfma_f32_16x16x32_f16 takes it as its B operand: lane
// 16 j + r holds row r, and its word w the columns 32 w + 8 j .. + 7, so no weight moves between lanes.  Next to the loads
// the instructions that turn nibbles into f16 set the pace: nine per eight weights.  0x6400 | q is the f16 1024 + q, with
// the nibble in bits 4..7 it is 1024 + 16 q; one packed add or multiply-add makes q - 8 of either, exactly.  (Taking q as
// the f16 subnormal q 2^-24 saves four of the nine, but the matrix unit aligns subnormal products by their exponent field
// and loses seven bits of them: 2e-6 instead of 1e-7 relative error.)
//
// x is f32.  It is split into two f16 parts (a power of two per row brings the largest finite |x| to 2^14..2^15), which
// stand in the 16 rows of the A operand: 8 rows of x in one product, so that a single one costs no more matrix instructions
// than eight.  A lane's results then belong to one row of W, whose scale it needs alone: the block's 64 scales (of groups of
// 32) are one 2-byte load per lane, which row swaps hand round.  Products are exact in f32, what the split leaves out is 2^-22 of a value (or 2^-39 of the
// row's largest, where that is more), a group's sum is multiplied by its scale in f32 and added up in f32.
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
constexpr int kXMost = 128 * 1024;                 // of x in LDS
constexpr size_t kQ4Lds = 158 * 1024;              // of the CU's 160 KB, the rest is the kernel's own
constexpr int kUnitTiles = 2;                      // tiles of a wave's unit where x is whole in LDS
constexpr int kAhead = 2;                          // blocks whose weights are in flight while one is multiplied (1: 43.5 instead of 41.7 us, 16 rows 61.5 / 53.2)
constexpr int kMaxExp = 127;                       // a power of two that is a float: x below 2^-112 keeps fewer bits
constexpr int kQ4Exp = 15;                         // a row's largest finite |x| goes to [2^14, 2^15)

struct Q4Params {
    const uint8_t * W;
    const _Float16 * scales;
    const float * x;
    float * y;
    const float * norm_w;
    int32_t out_dim, in_dim, rows;
    int32_t n_tiles, n_units;                     // tiles of y, and how many units of work they make
    int32_t wt, wk;                               // waves over units and over columns: wt * wk = kQ4Waves
    int32_t epilogue;
    float eps;
};

// Waves that share a row of x when its factor is computed.
__host__ __device__ inline int row_parts(int rows) { return rows <= 1 ? 8 : rows <= 2 ? 4 : rows <= 4 ? 2 : 1; }

// RMSNorm's factor from a row's sum of squares.  A mean past f32's range (x of 2e19 and more) goes there by 2^-140, where eps
// is nothing beside it, and its root's half comes back.
__device__ inline float norm_factor(double sum, int dim, float eps) {
    const double mean = sum / dim;
    const bool past = mean > 3e38;
    const float f = 1.0f / sqrtf(past ? static_cast<float>(mean * 0x1p-140) : static_cast<float>(mean) + eps);
    return past ? f * 0x1p-70f : f;
}

// 8 nibbles of a word as q - 8 in column order (column e lies in bits 4 (e / 2) + 16 (e % 2)).
struct Unpack {
    uint32_t low, high, magic;
    h2 off, off16, sixteenth;
    __device__ inline Unpack() {
        low = 0x000f000fu;
        high = 0x00f000f0u;
        magic = 0x64006400u;
        // masks in registers: an instruction takes one constant that is none, and there are two
        asm("" : "+v"(low), "+v"(high));
        asm("" : "+s"(magic));
        off = h2{static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
        off16 = h2{static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
        sixteenth = h2{static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    }
    __device__ inline h8 operator()(uint32_t w) const {
        const uint32_t v = w >> 8;
        const h2 a = __builtin_bit_cast(h2, (w & low) | magic) + off;
        const h2 b = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & high) | magic), sixteenth, off16);
        const h2 c = __builtin_bit_cast(h2, (v & low) | magic) + off;
        const h2 d = __builtin_elementwise_fma(__builtin_bit_cast(h2, (v & high) | magic), sixteenth, off16);
        return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
};

// 4 neighbouring values of an x row, times the row's power of two (no product is rounded here), as the two f16 parts.
// inf: the row holds an infinity, whose second part is 0 instead of inf - inf.
__device__ inline void split_x(f4 v, float unit, bool inf, _Float16 * to) {
    h4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float s = v[e] * unit;
        hi[e] = static_cast<_Float16>(s);
        lo[e] = static_cast<_Float16>(s - static_cast<float>(hi[e]));
        if (inf && fabsf(s) == INFINITY) lo[e] = static_cast<_Float16>(0.0f);
    }
    *reinterpret_cast<h4 *>(to) = hi;
    *reinterpret_cast<h4 *>(to + 32) = lo;
}

// The A operand of lanes c16 and c16 + 8 of a row from four scaled values each: the first parts of the eight in one, the second
// parts in the other.  Scaling was by a power of two, so that no product is rounded here.
__device__ inline h8 split_pair(f4 v, bool inf, bool second) {
    h4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = static_cast<_Float16>(v[e]);
        lo[e] = static_cast<_Float16>(v[e] - static_cast<float>(hi[e]));
    }
    if (__builtin_expect(inf, 0)) {
        asm volatile("");                                         // a branch, not a selection per value
#pragma unroll
        for (int e = 0; e < 4; ++e) lo[e] = fabsf(v[e]) == INFINITY ? static_cast<_Float16>(0.0f) : lo[e];
    }
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const u2 h = __builtin_bit_cast(u2, hi), l = __builtin_bit_cast(u2, lo);
    const u2 send = second ? h : l;                               // to the other lane
    const u2 got = {__float_as_uint(row_ror8(__uint_as_float(send[0]))), __float_as_uint(row_ror8(__uint_as_float(send[1])))};
    const u4 a = second ? u4{got[0], got[1], l[0], l[1]} : u4{h[0], h[1], got[0], got[1]};
    return __builtin_bit_cast(h8, a);
}

// The scales of a block's groups in every lane, from one value per lane: groups of 32 lie in the four rows of 16 lanes, groups
// of 64 in the first two (and again in the others).
template <int GS>
__device__ inline void spread_scales(float v, float (&d)[4 >> GS]) {
    const uint32_t x = __float_as_uint(v);
    if constexpr (GS == 2) {
        d[0] = v;
    } else {
        const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);   // rows 0 0 2 2 and 1 1 3 3
        if constexpr (GS == 1) {
            d[0] = __uint_as_float(a[0]);
            d[1] = __uint_as_float(a[1]);
        } else {
            const auto even = __builtin_amdgcn_permlane32_swap(a[0], a[0], false, false);
            const auto odd = __builtin_amdgcn_permlane32_swap(a[1], a[1], false, false);
            d[0] = __uint_as_float(even[0]);
            d[1] = __uint_as_float(odd[0]);
            d[2] = __uint_as_float(even[1]);
            d[3] = __uint_as_float(odd[1]);
        }
    }
}

// x row r of a block of 8 stands in rows (r % 2) 4 + r / 2 of the A operand, its second part 8 rows on: a lane's result i
// belongs to x row 2 i + (lane / 16) % 2, so that up to 2 rows need the first result alone.
// NB: blocks of 8 x rows.  NI: results of a lane that count (1 or 4).  A wave's unit is two tiles, with SwiGLU gate and up.  GS: groups of 32 << GS columns.  All of x lies in LDS.
template <int NB, int NI, bool SWIGLU, int GS>
__global__ __launch_bounds__(kQ4Threads, 2) void gemv_q4_kernel(Q4Params p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    _Float16 * sx = reinterpret_cast<_Float16 *>(lds);            // [in_dim / 32][row][part][32]
    __shared__ float s_factor[kQ4MaxRows];                        // RMSNorm factor of each row
    __shared__ int s_exp[kQ4MaxRows];                             // and the power of two of its x
    __shared__ double s_sum[kQ4Waves];                            // of a row's parts
    __shared__ float s_max[kQ4Waves];                             // a sign: an infinity among them
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    const int wk = wave % p.wk, wt = wave / p.wk;
    const int n_kb = p.in_dim / kTileCols;
    // units go to the waves of all workgroups in turn, so that every CU gets as many
    const int unit_step = static_cast<int>(gridDim.x) * p.wt;
    const int unit0 = wt * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);

    // weights and scales of the next kAhead blocks are in flight, the first ones while x is prepared; behind its last block a
    // wave loads that one again, so that no branch makes it wait for all
    constexpr int kGroups = 4 >> GS;                              // of a block
    u4 w[kAhead][kUnitTiles];
    _Float16 d[kAhead][kUnitTiles];
    const int n_it = (n_kb + p.wk * kAhead - 1) / (p.wk * kAhead) * kAhead;   // a wave's blocks of a unit, the last ones perhaps idle
    const uint32_t w_lane = lane * 16, d_lane = (lane & (kGroups * kTileRows - 1)) * 2;
    int f_unit = unit0, f_it = 0;
    auto fetch = [&](int slot) {
        const int kb = min(wk + f_it * p.wk, n_kb - 1), unit = f_unit < p.n_units ? f_unit : min(unit0, p.n_units - 1);
#pragma unroll
        for (int t = 0; t < kUnitTiles; ++t) {
            const int tile = SWIGLU ? unit + t * p.n_tiles : min(unit * kUnitTiles + t, p.n_tiles - 1);
            const int64_t at = static_cast<int64_t>(tile) * n_kb + kb;
            const char * wb = reinterpret_cast<const char *>(p.W) + at * (kWave * 16);
            const char * db = reinterpret_cast<const char *>(p.scales) + at * (kGroups * kTileRows * 2);
            // a matrix of more than 1024 tiles past the caches, which hold it no better (151936 x 2048: 8 rows 41.7 instead of 42.3 us, one row alike)
            w[slot][t] = __builtin_nontemporal_load(reinterpret_cast<const u4 *>(wb + w_lane));
            d[slot][t] = *reinterpret_cast<const _Float16 *>(db + d_lane);
        }
        if (++f_it == n_it) {
            f_it = 0;
            f_unit += unit_step;
        }
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) fetch(u);

    // Sum of squares and largest |x| of each row: the 8 waves share up to 8 rows, each taking a part of a row whose loads are
    // in flight together.  A workgroup that holds all of x writes its parts from those registers.
    const f4 * nw = reinterpret_cast<const f4 *>(p.norm_w);
    const int parts = row_parts(p.rows);
    const int part = wave % parts, n4 = p.in_dim >> 2, step = parts * kWave;
    const int cols = 2 * p.rows;
    constexpr int kPer = 8;
    f4 v[kPer];
    double ss;
    float mx;
    bool inf;
    auto read_part = [&](int r) {
        const f4 * x = reinterpret_cast<const f4 *>(p.x + static_cast<int64_t>(r) * p.in_dim);
        ss = 0.0;
        mx = 0.0f;
        // rounds that lie behind the row for the whole wave load nothing
        for (int k0 = part * kWave; k0 < n4; k0 += kPer * step) {
            f4 g[kPer];
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                if (k0 + u * step >= n4) break;
                const int at = min(k0 + lane + u * step, n4 - 1);
                v[u] = x[at];
                if (nw) g[u] = nw[at];
            }
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                if (k0 + u * step >= n4) break;
                if (k0 + lane + u * step >= n4) continue;
                if (nw) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ss += static_cast<double>(v[u][e]) * v[u][e];
                        v[u][e] *= g[u][e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(v[u][e]));
            }
        }
        ss = nw ? wave_sum_d_all(ss) : 0.0;
        mx = wave_max_all(mx);
        inf = mx == INFINITY;
        if (__builtin_expect(inf, 0)) {                           // rare: the largest of what is finite
            mx = 0.0f;
            for (int k = part * kWave + lane; k < n4; k += step) {
                const f4 a = nw ? x[k] * nw[k] : x[k];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (fabsf(a[e]) < INFINITY) mx = fmaxf(mx, fabsf(a[e]));
                }
            }
            mx = wave_max_all(mx);
        }
    };
    auto finish_row = [&](int r) {
        // RMSNorm's factor is one of the result: the factor of a small row times its power of two is no float
        const int ex = mx > 0.0f ? min(kQ4Exp - __builtin_amdgcn_frexp_expf(mx), kMaxExp) : 0;
        const float unit = ldexpf(1.0f, ex);
        if (lane == 0 && part == 0) {
            s_factor[r] = p.norm_w ? norm_factor(ss, p.in_dim, p.eps) : 1.0f;
            s_exp[r] = ex;
        }
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int k = part * kWave + lane + u * step;
            if (k < n4) split_x(v[u], unit, inf, sx + ((k >> 3) * cols + 2 * r) * 32 + (k & 7) * 4);
        }
    };
    if (parts > 1) {                                              // one row per wave at most, parts of it in several
        const int r = wave / parts;
        if (r < p.rows) read_part(r);
        if (r < p.rows && lane == 0) {
            s_sum[wave] = ss;
            s_max[wave] = inf ? -mx : mx;
        }
        __syncthreads();
        if (r < p.rows) {
            ss = 0.0;
            mx = 0.0f;
            inf = false;
            for (int i = r * parts; i < (r + 1) * parts; ++i) {
                ss += s_sum[i];
                mx = fmaxf(mx, fabsf(s_max[i]));
                inf = inf || __float_as_uint(s_max[i]) >> 31;
            }
            finish_row(r);
        }
    } else {
        for (int r = wave; r < p.rows; r += kQ4Waves) {
            read_part(r);
            finish_row(r);
        }
    }
    __syncthreads();

    int arow[NB];
    const int a8 = c16 & 7, xr = (a8 & 3) * 2 + (a8 >> 2);        // the x row of the A row c16
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) arow[nb] = (2 * min(nb * 8 + xr, p.rows - 1) + (c16 >> 3)) * 32 + g4 * 8;
    float acc[kUnitTiles][NB][NI];
    auto clear = [&]() {
#pragma unroll
        for (int t = 0; t < kUnitTiles; ++t) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int i = 0; i < NI; ++i) acc[t][nb][i] = 0.0f;
            }
        }
    };
    const Unpack unpack;
    auto block = [&](int slot, int kb_in_lds, bool counts) {
        const _Float16 * xb = sx + static_cast<int64_t>(kb_in_lds) * 4 * cols * 32;
        f4 group[kUnitTiles][NB];
        float dg[kUnitTiles][kGroups];
#pragma unroll
        for (int t = 0; t < kUnitTiles; ++t) spread_scales<GS>(static_cast<float>(d[slot][t]), dg[t]);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const bool first = (s & ((1 << GS) - 1)) == 0, last = ((s + 1) & ((1 << GS) - 1)) == 0;
            h8 a[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) a[nb] = *reinterpret_cast<const h8 *>(xb + s * cols * 32 + arow[nb]);
#pragma unroll
            for (int t = 0; t < kUnitTiles; ++t) {
                const h8 b = unpack(w[slot][t][s]);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const f4 c = first ? f4{0.0f, 0.0f, 0.0f, 0.0f} : group[t][nb];
                    group[t][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[nb], b, c, 0, 0, 0);
                    if (last && counts) {
#pragma unroll
                        for (int i = 0; i < NI; ++i) acc[t][nb][i] = fmaf(group[t][nb][i], dg[t][s >> GS], acc[t][nb][i]);
                    }
                }
            }
        }
        fetch(slot);
    };
    // results of a unit: lane c16 + 16 g4 holds row c16 of the tile, the two parts of x lie 32 lanes apart
    auto store = [&](int unit) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = nb * 8 + 2 * i + (g4 & 1);
                float v[kUnitTiles];
#pragma unroll
                for (int t = 0; t < kUnitTiles; ++t) v[t] = acc[t][nb][i] + __shfl_xor(acc[t][nb][i], 32, kWave);
                if (g4 >= 2 || r >= p.rows) continue;
#pragma unroll
                for (int t = 0; t < (SWIGLU ? 1 : kUnitTiles); ++t) {
                    const int o = (SWIGLU ? unit : unit * kUnitTiles + t) * kTileRows + c16;
                    if (o >= p.out_dim) continue;                 // rows and tiles behind the last
                    float * y = p.y + static_cast<int64_t>(r) * p.out_dim + o;
                    float out = ldexpf(v[t] * s_factor[r], -s_exp[r]);
                    if constexpr (SWIGLU) out = out / (1.0f + expf(-out)) * ldexpf(v[1] * s_factor[r], -s_exp[r]);
                    *y = p.epilogue == kEpiAccumOp ? *y + out : out;
                }
            }
        }
    };
    // the waves of a unit's columns add up in LDS, in order, behind the x that the next unit takes again
    float * sa = reinterpret_cast<float *>(lds + static_cast<size_t>(p.in_dim) * p.rows * 4);
    auto join = [&]() {
        constexpr int kVals = kUnitTiles * NB * NI;
        __syncthreads();                                          // what lay there has been read
        if (wk > 0) {
#pragma unroll
            for (int t = 0; t < kUnitTiles; ++t) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int i = 0; i < NI; ++i) sa[((wt * (p.wk - 1) + wk - 1) * kVals + (t * NB + nb) * NI + i) * kWave + lane] = acc[t][nb][i];
                }
            }
        }
        __syncthreads();
        for (int k = 0; k < p.wk - 1 && wk == 0; ++k) {
#pragma unroll
            for (int t = 0; t < kUnitTiles; ++t) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int i = 0; i < NI; ++i) acc[t][nb][i] += sa[((wt * (p.wk - 1) + k) * kVals + (t * NB + nb) * NI + i) * kWave + lane];
                }
            }
        }
    };
    // all waves of the workgroup go as many rounds: the join has barriers
    const int rounds = (p.n_units + unit_step - 1) / unit_step;
    for (int round = 0; round < rounds; ++round) {
        const int unit = unit0 + round * unit_step;
        clear();
        for (int it = 0; it < n_it; it += kAhead) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int kb = wk + (it + u) * p.wk;
                block(u, min(kb, n_kb - 1), kb < n_kb);
            }
        }
        if (p.wk > 1) join();
        if (wk == 0 && unit < p.n_units) store(unit);
    }
}

// The form for an x that does not fit in LDS, or that only a few tiles would share: a workgroup is 8 rows of x and NU tiles (with
// SwiGLU: of gate and as many of up), its 8 waves share the columns, and a wave reads the x of its own blocks as the A operand, with
// no barrier before the end.  Its lane c16 holds x row r's columns 8 g4 .. + 3 of a step and lane c16 + 8 those .. + 7; each splits its
// four and the two exchange the parts, so that one has the first parts of all eight and the other the second.  One pass over
// x: a wave keeps a power of two per row that fits what it has seen and rescales its sums when that falls; the sum of squares
// comes along, and its factor is one of the result.  What bounds it is the arithmetic on x, 9 (with the norm 12)
// instructions a value: the rows of more than 8 are workgroups of their own, which read W again, from L2 (2048 x 6144, 16
// rows: 10.2 us, as one workgroup's 16.0), and tiles go together where there are workgroups enough without.
template <int NU, bool SWIGLU, int GS>
__global__ __launch_bounds__(kQ4Threads, 2) void gemv_q4_rows_kernel(Q4Params p) {
    constexpr int TW = SWIGLU ? 2 * NU : NU, kRows = 8, kGroups = 4 >> GS, kVals = TW * 4;   // tile t: with SwiGLU of the pair t / 2
    __shared__ float sa[kQ4Waves][kVals][kWave];
    __shared__ double s_sum[kQ4Waves][kRows];
    __shared__ int s_exp[kQ4Waves][kRows];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    const bool second = c16 >= 8;
    const int a8 = c16 & 7, xr = (a8 & 3) * 2 + (a8 >> 2);        // the x row of the A row c16, as in the form above
    const int n_kb = p.in_dim / kTileCols, unit = blockIdx.x;
    const int row0 = blockIdx.y * kRows, rows = min(kRows, p.rows - row0);
    const float * xrow = p.x + static_cast<int64_t>(row0 + min(xr, rows - 1)) * p.in_dim + g4 * 8 + (second ? 4 : 0);
    const float * nrow = p.norm_w ? p.norm_w + g4 * 8 + (second ? 4 : 0) : nullptr;

    u4 w[TW];
    _Float16 d[TW];
    f4 x[4], g[4];
    auto fetch = [&](int kb) {
#pragma unroll
        for (int t = 0; t < TW; ++t) {
            const int tile = SWIGLU ? min(unit * NU + t / 2, p.n_tiles - 1) + (t & 1) * p.n_tiles : min(unit * NU + t, p.n_tiles - 1);
            const int64_t at = static_cast<int64_t>(tile) * n_kb + kb;
            w[t] = reinterpret_cast<const u4 *>(p.W)[at * kWave + lane];
            d[t] = p.scales[at * kGroups * kTileRows + (lane & (kGroups * kTileRows - 1))];
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            x[s] = *reinterpret_cast<const f4 *>(xrow + kb * kTileCols + s * 32);
            if (nrow) g[s] = *reinterpret_cast<const f4 *>(nrow + kb * kTileCols + s * 32);
        }
    };
    float acc[TW][4];
#pragma unroll
    for (int t = 0; t < TW; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = 0.0f;
    }
    double ss = 0.0;
    int ex = kMaxExp;
    const Unpack unpack;
    if (wave < n_kb) fetch(wave);
    for (int kb = wave; kb < n_kb; kb += kQ4Waves) {
        if (nrow) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    ss += static_cast<double>(x[s][e]) * x[s][e];
                    x[s][e] *= g[s][e];
                }
            }
        }
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(x[s][e]));
        }
        mx = column_max(fmaxf(mx, row_ror8(mx)));
        const bool inf = __ballot(mx == INFINITY) != 0;
        if (__builtin_expect(inf, 0)) {                           // rare: the largest of what is finite
            mx = 0.0f;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fabsf(x[s][e]) < INFINITY ? fmaxf(mx, fabsf(x[s][e])) : mx;
            }
            mx = column_max(fmaxf(mx, row_ror8(mx)));
        }
        const int to = mx > 0.0f ? min(ex, kQ4Exp - __builtin_amdgcn_frexp_expf(mx)) : ex;
        if (__ballot(to < ex) != 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int by = __shfl(to - ex, 4 * (g4 & 1) + i, kWave);
#pragma unroll
                for (int t = 0; t < TW; ++t) acc[t][i] = ldexpf(acc[t][i], by);
            }
            ex = to;
        }
        const float factor = ldexpf(1.0f, ex);
        h8 a[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) a[s] = split_pair(x[s] * factor, inf, second);
        u4 wb[TW];
        float dg[TW][kGroups];
#pragma unroll
        for (int t = 0; t < TW; ++t) {
            wb[t] = w[t];
            spread_scales<GS>(static_cast<float>(d[t]), dg[t]);
        }
        fetch(min(kb + kQ4Waves, n_kb - 1));                      // behind its last block a wave loads one that nobody uses
        f4 group[TW];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const bool first = (s & ((1 << GS) - 1)) == 0, last = ((s + 1) & ((1 << GS) - 1)) == 0;
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                const f4 c = first ? f4{0.0f, 0.0f, 0.0f, 0.0f} : group[t];
                group[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[s], unpack(wb[t][s]), c, 0, 0, 0);
                if (last) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(group[t][i], dg[t][s >> GS], acc[t][i]);
                }
            }
        }
    }
    // the waves' sums meet at the smallest of their powers of two, and add up in order
#pragma unroll
    for (int m = 8; m < kWave; m <<= 1) ss += __shfl_xor(ss, m, kWave);
    if (lane < 8) {
        s_sum[wave][xr] = ss;
        s_exp[wave][xr] = ex;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 2 * i + (g4 & 1);
        int least = s_exp[0][r];
#pragma unroll
        for (int k = 1; k < kQ4Waves; ++k) least = min(least, s_exp[k][r]);
        const int by = least - s_exp[wave][r];
#pragma unroll
        for (int t = 0; t < TW; ++t) sa[wave][t * 4 + i][lane] = ldexpf(acc[t][i], by);
    }
    __syncthreads();
    constexpr int kOf = SWIGLU ? 2 : 1;                           // sums of a result
    for (int j = wave; j < NU * 4; j += kQ4Waves) {
        const int n = j >> 2, i = j & 3;
        float v[kOf];
#pragma unroll
        for (int t = 0; t < kOf; ++t) {
            v[t] = 0.0f;
#pragma unroll
            for (int k = 0; k < kQ4Waves; ++k) v[t] += sa[k][(n * kOf + t) * 4 + i][lane];
            v[t] += __shfl_xor(v[t], 32, kWave);
        }
        const int r = 2 * i + (g4 & 1), o = (unit * NU + n) * kTileRows + c16;
        if (g4 >= 2 || r >= rows || o >= p.out_dim) continue;     // rows and tiles behind the last
        double sum = 0.0;
        int least = kMaxExp;
#pragma unroll
        for (int k = 0; k < kQ4Waves; ++k) {
            sum += s_sum[k][r];
            least = min(least, s_exp[k][r]);
        }
        const float f = p.norm_w ? norm_factor(sum, p.in_dim, p.eps) : 1.0f;
        float * y = p.y + static_cast<int64_t>(row0 + r) * p.out_dim + o;
        float out = ldexpf(v[0] * f, -least);
        if constexpr (SWIGLU) out = out / (1.0f + expf(-out)) * ldexpf(v[1] * f, -least);
        *y = p.epilogue == kEpiAccumOp ? *y + out : out;
    }
}

// The same for a single x: its 8 rows of the A operand are 8 blocks of columns instead, split at once, so that the arithmetic on x is an
// eighth; the product with W's block j gives its result in row j, and the others, of unlike blocks, are dropped.  All of a wave's
// weights are in flight at once.  us with the form above: 2048 x 6144 6.1 / 7.9, 12288 gate|up rows 7.1 / 8.5, 4096 x 2048 4.9 / 5.3.
template <int NU, bool SWIGLU, int GS>
__global__ __launch_bounds__(kQ4Threads, 2) void gemv_q4_token_kernel(Q4Params p) {
    constexpr int TW = SWIGLU ? 2 * NU : NU, kGroups = 4 >> GS, kBlocks = 8;
    __shared__ float sa[kQ4Waves][TW][kWave];
    __shared__ double s_sum[kQ4Waves];
    __shared__ int s_exp[kQ4Waves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4, a8 = c16 & 7;
    const bool second = c16 >= 8;
    const int n_kb = p.in_dim / kTileCols, unit = blockIdx.x;
    const int col = g4 * 8 + (second ? 4 : 0);
    float acc[TW];
#pragma unroll
    for (int t = 0; t < TW; ++t) acc[t] = 0.0f;
    double ss = 0.0;
    int ex = kMaxExp;
    const Unpack unpack;
    for (int kb0 = wave; kb0 < n_kb; kb0 += kBlocks * kQ4Waves) {
        // every load of the 8 blocks at once; behind the last block it is that one again
        const int mine = kb0 + a8 * kQ4Waves;
        const bool counts = mine < n_kb;
        const int at = min(mine, n_kb - 1) * kTileCols + col;
        f4 x[4], g[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            x[s] = *reinterpret_cast<const f4 *>(p.x + at + s * 32);
            if (p.norm_w) g[s] = *reinterpret_cast<const f4 *>(p.norm_w + at + s * 32);
        }
        u4 w[kBlocks][TW];
        _Float16 d[kBlocks][TW];
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
            if (kb0 + j * kQ4Waves >= n_kb) break;                // uniform for the wave
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                const int tile = SWIGLU ? min(unit * NU + t / 2, p.n_tiles - 1) + (t & 1) * p.n_tiles : min(unit * NU + t, p.n_tiles - 1);
                const int64_t b = static_cast<int64_t>(tile) * n_kb + kb0 + j * kQ4Waves;
                w[j][t] = reinterpret_cast<const u4 *>(p.W)[b * kWave + lane];
                d[j][t] = p.scales[b * kGroups * kTileRows + (lane & (kGroups * kTileRows - 1))];
            }
        }
        if (p.norm_w) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (counts) ss += static_cast<double>(x[s][e]) * x[s][e];
                    x[s][e] *= g[s][e];
                }
            }
        }
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(x[s][e]));
        }
        mx = wave_max_all(mx);
        const bool inf = mx == INFINITY;
        if (__builtin_expect(inf, 0)) {                           // rare: the largest of what is finite
            mx = 0.0f;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fabsf(x[s][e]) < INFINITY ? fmaxf(mx, fabsf(x[s][e])) : mx;
            }
            mx = wave_max_all(mx);
        }
        const int to = mx > 0.0f ? min(ex, kQ4Exp - __builtin_amdgcn_frexp_expf(mx)) : ex;
#pragma unroll
        for (int t = 0; t < TW; ++t) acc[t] = ldexpf(acc[t], to - ex);
        ex = to;
        const float factor = ldexpf(1.0f, ex);
        h8 a[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) a[s] = split_pair(x[s] * factor, inf, second);
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
            if (kb0 + j * kQ4Waves >= n_kb) break;
            const bool row = (g4 & 1) == j / 4;                   // this lane's results are rows 4 (g4 % 2) .. + 3, in one part of x
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                float dg[kGroups];
                spread_scales<GS>(static_cast<float>(d[j][t]), dg);
                f4 group;
                float sum = 0.0f;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const bool first = (s & ((1 << GS) - 1)) == 0, last = ((s + 1) & ((1 << GS) - 1)) == 0;
                    const f4 c = first ? f4{0.0f, 0.0f, 0.0f, 0.0f} : group;
                    group = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[s], unpack(w[j][t][s]), c, 0, 0, 0);
                    if (last) sum = fmaf(group[j & 3], dg[s >> GS], sum);
                }
                acc[t] += row ? sum : 0.0f;
            }
        }
    }
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) ss += __shfl_xor(ss, m, kWave);   // every x is in one lane
    if (lane == 0) {
        s_sum[wave] = ss;
        s_exp[wave] = ex;
    }
    __syncthreads();
    int least = s_exp[0];
    double sum = s_sum[0];
#pragma unroll
    for (int k = 1; k < kQ4Waves; ++k) {
        least = min(least, s_exp[k]);
        sum += s_sum[k];
    }
#pragma unroll
    for (int t = 0; t < TW; ++t) sa[wave][t][lane] = ldexpf(acc[t], least - ex);
    __syncthreads();
    constexpr int kOf = SWIGLU ? 2 : 1;                           // sums of a result
    for (int n = wave; n < NU; n += kQ4Waves) {
        float v[kOf];
#pragma unroll
        for (int t = 0; t < kOf; ++t) {
            v[t] = 0.0f;
#pragma unroll
            for (int k = 0; k < kQ4Waves; ++k) v[t] += sa[k][n * kOf + t][lane];
            v[t] += __shfl_xor(v[t], 16, kWave);
            v[t] += __shfl_xor(v[t], 32, kWave);
        }
        const int o = (unit * NU + n) * kTileRows + c16;
        if (g4 > 0 || o >= p.out_dim) continue;
        const float f = p.norm_w ? norm_factor(sum, p.in_dim, p.eps) : 1.0f;
        float out = ldexpf(v[0] * f, -least);
        if constexpr (SWIGLU) out = out / (1.0f + expf(-out)) * ldexpf(v[1] * f, -least);
        p.y[o] = p.epilogue == kEpiAccumOp ? p.y[o] + out : out;
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

int launch_q4_kernel(void (*kernel)(Q4Params), const Q4Params & p, dim3 blocks, size_t lds, hipStream_t stream) {
    if (lds > 32 * 1024) {
        QA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
    }
    hipLaunchKernelGGL(kernel, blocks, dim3(kQ4Threads), lds, stream, p);
    QA_LAUNCH_CHECK("4-bit matrix-vector kernel");
    return QA_OK;
}

// How the waves divide the work where x is whole in LDS.  Units alone rarely fill the GPU evenly (9496 tiles over 4096 waves are
// two rounds and a bit), so a unit's columns are shared by up to 8 waves, the more of them the fewer rows x has to be read
// for: a tile's partial sums then meet in LDS.  No more workgroups run than are resident.
// Measured with 1 / 2 / 4 / 8 waves per unit, 151936 x 2048: one row 56 / 43 / 37.6 / 38.2 us, 8 rows 57 / 46 / 42.0 / 43.5, 16 rows
// 56 / 54 / 63 / 77 (one card; the same call differs by 6% between cards, 8 rows 39 to 42).
template <int NB, int NI, bool SWIGLU, int GS>
int launch_q4(Q4Params p, hipStream_t stream) {
    p.n_units = SWIGLU ? p.n_tiles : (p.n_tiles + kUnitTiles - 1) / kUnitTiles;
    const int n_kb = p.in_dim / kTileCols;
    const int64_t waves = NB == 1 ? 16384 : NB == 2 ? 8192 : 4096;
    const size_t join = static_cast<size_t>(kUnitTiles) * NB * NI * kWave * 4, x_bytes = static_cast<size_t>(p.in_dim) * p.rows * 4;
    p.wk = 1;
    while (p.wk < kQ4Waves && p.wk * 2 <= n_kb && static_cast<int64_t>(p.n_units) * p.wk < waves &&
           x_bytes + (kQ4Waves - kQ4Waves / (p.wk * 2)) * join <= kQ4Lds) {
        p.wk *= 2;
    }
    p.wt = kQ4Waves / p.wk;
    const int units = (p.n_units + p.wt - 1) / p.wt;
    const size_t lds = x_bytes + p.wt * (p.wk - 1) * join;
    const int blocks = std::min(units, lds <= 80 * 1024 - 1024 ? 512 : 256);
    return launch_q4_kernel(&gemv_q4_kernel<NB, NI, SWIGLU, GS>, p, dim3(blocks), lds, stream);
}

int row_groups(int rows) { return (rows + 7) / 8; }

template <bool SWIGLU, int GS>
int launch_q4_own(const Q4Params & p, hipStream_t stream) {
    const int parts = row_groups(p.rows);
    // one workgroup per CU, and the fewest tiles that bring it to that: a workgroup splits its x once for all of them.  256 tiles, 32 rows
    // in 1 / 2 / 4 16.4 / 10.4 / 8.8 us; 384 pairs, 8 rows 11.1 / 9.1 / 11.9.
    int nu = 1;
    while (nu < 4 && (p.n_tiles + nu - 1) / nu * parts > 256) ++nu;
    const dim3 blocks((p.n_tiles + nu - 1) / nu, parts);
    if (p.rows == 1 && nu * (SWIGLU ? 2 : 1) <= 4) {              // more tiles' blocks than that pass a lane's registers
        if (nu == 1) return launch_q4_kernel(&gemv_q4_token_kernel<1, SWIGLU, GS>, p, blocks, 0, stream);
        if (nu == 2) return launch_q4_kernel(&gemv_q4_token_kernel<2, SWIGLU, GS>, p, blocks, 0, stream);
        if constexpr (!SWIGLU) return launch_q4_kernel(&gemv_q4_token_kernel<4, SWIGLU, GS>, p, dim3((p.n_tiles + 3) / 4), 0, stream);
    }
    if (nu == 1) return launch_q4_kernel(&gemv_q4_rows_kernel<1, SWIGLU, GS>, p, blocks, 0, stream);
    if (nu == 2) return launch_q4_kernel(&gemv_q4_rows_kernel<2, SWIGLU, GS>, p, blocks, 0, stream);
    if (nu == 3) return launch_q4_kernel(&gemv_q4_rows_kernel<3, SWIGLU, GS>, p, blocks, 0, stream);
    return launch_q4_kernel(&gemv_q4_rows_kernel<4, SWIGLU, GS>, p, blocks, 0, stream);
}

// Whether x fits in LDS and a wave's share of a row in its registers.  Behind that limit a vocabulary's x is split again for every
// four of its tiles: 151936 x 2048 / 2176 columns, 4 rows 36 / 46 us, 8 rows 40 / 81, 16 rows 52 / 149, 32 rows 103 / 284; 4096 columns,
// 4 rows 66, 8 rows 117.
bool whole_x(int rows, int in_dim) {
    return in_dim <= 2048 * row_parts(rows) && static_cast<int64_t>(rows) * in_dim * 4 <= kXMost;
}

template <bool SWIGLU, int GS>
int launch_q4_shared(const Q4Params & p, hipStream_t stream) {
    if (p.rows <= 2) return launch_q4<1, 1, SWIGLU, GS>(p, stream);
    if (p.rows <= 8) return launch_q4<1, 4, SWIGLU, GS>(p, stream);
    if (p.rows <= 16) return launch_q4<2, 4, SWIGLU, GS>(p, stream);
    return launch_q4<4, 4, SWIGLU, GS>(p, stream);
}

template <bool SWIGLU, int GS>
int launch_q4_rows(const Q4Params & p, hipStream_t stream) {
    // Up to 1024 tiles every wave splits the x of its own columns, us against x in LDS: 128 tiles of 2048 columns 1 / 8 / 32 rows 4.4 / 5.4 /
    // 5.9 against 5.0 / 6.6 / 19.2, 256 tiles 4.9 / 6.0 / 8.7 against 5.4 / 7.4 / 21.7, 1024 tiles 7.3 / 9.3 / 30.6 against 8.4 / 12.7 /
    // 33.4, 384 pairs of tiles (12288 gate|up rows) 7.1 / 8.8 / 22.1 against 8.1 / 12.2 / 33.8; 2048 tiles 15.7 / 17.4 / 59.7
    // against 12.1 / 16.6 / 48.3, and 1024 pairs of 1024 columns 24 rows 24.1 against 21.5.
    const int at_once = whole_x(p.rows, p.in_dim) ? p.rows : std::min(p.rows, 16);   // of more, 16 rows at a time: W is read twice
    const bool few = p.n_tiles <= 1024 && (!SWIGLU || p.n_tiles * row_groups(p.rows) <= 2048);
    if (few || !whole_x(at_once, p.in_dim)) return launch_q4_own<SWIGLU, GS>(p, stream);
    Q4Params part = p;
    for (int r = 0; r < p.rows; r += at_once) {
        part.rows = std::min(at_once, p.rows - r);
        if (const int rc = launch_q4_shared<SWIGLU, GS>(part, stream); rc != QA_OK) return rc;
        part.x += static_cast<int64_t>(at_once) * p.in_dim;
        part.y += static_cast<int64_t>(at_once) * p.out_dim;
    }
    return QA_OK;
}

template <int GS>
int launch_q4_tiles(const Q4Params & p, hipStream_t stream) {
    return p.epilogue == kEpiSwigluOp ? launch_q4_rows<true, GS>(p, stream) : launch_q4_rows<false, GS>(p, stream);
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
    p.n_tiles = (out_dim + kTileRows - 1) / kTileRows;
    p.epilogue = epilogue;
    p.eps = eps;
    switch (group) {
        case 32: return launch_q4_tiles<0>(p, as_stream(stream));
        case 64: return launch_q4_tiles<1>(p, as_stream(stream));
        default: return launch_q4_tiles<2>(p, as_stream(stream));
    }
}
