// Attention of each sequence's new tokens over a K/V cache in pages: causal, or by a tree's masks.
//
//   o_t = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q_t . k_j - m_t),   j <= n_past + t on a page that exists
//                                                       (trees: j < n_past, and the new tokens of row t's mask)
//
// in one pass over the keys with a running maximum m and sum (the accumulators are rescaled when m grows).  The query
// heads of a KV head and the tokens of a sequence are columns of the same products: column c of a tile is token c / group
// and head c % group, so one token of 2 heads and a chunk of a thousand run the same code, in three shapes: a workgroup
// takes 16 columns (8 in the packed form) or 32 and its 4 or 8 waves share the keys (attn_rows; attn_wide: trees and 8 bits), or
// 128, a quarter per wave, and the waves share K and V (attn_tile, long causal chunks on f16 pages).  A batch with short and
// long sequences is one launch.
//
// f16 pages on v_mfma_f32_16x16x32_f16: q and p are f32, split into two f16 parts each (a power of two per column brings
// the largest |q| to 2^14..2^15, p is scaled by 2^6, so the second part keeps its bits); K and V are exact f16.  What the
// parts leave out is 2^-22 of a value, the result is as near to 64 bits as f32 products are.  Up to 8 columns carry both
// parts in one 16-column product (PACK), for decode steps.  f32 pages on v_mfma_f32_16x16x4_f32, whose products are f32.
// Pages of 8 bits: the integers are exact f16, one conversion each; scores are multiplied by their key's scale, which is the
// product with the dequantised K, and V's scales go into the probabilities before these are split (weighted_step).  What bounds them is the
// instructions of the conversions (128 of the 330 of a step of 32 keys by 32 columns, which has 64 products) besides memory.
//
// Operands.  S^T = K Q^T takes K rows as they lie: lane l holds key l % 16.  attn_rows and attn_wide bring K's rows into LDS as they
// lie and read operands there (KStep); V goes straight from memory into registers.  The result of S^T leaves 4 keys of a
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
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazyLog2 = 8.0f;    // the reference maximum follows when it is behind by more than 2^8
constexpr float kShiftLog2 = 6.0f;   // p is scaled by 2^6: at most 2^14 in f16, and its second part stays normal
constexpr int kQExp = 15;            // a column's largest |q| goes to [2^14, 2^15)
constexpr int kMaxSplits = 64;       // key ranges whose results the joining kernel adds, one lane each
constexpr int kWaves = 4, kThreads = kWaves * kWave;
// Sequences of few columns: a workgroup holds all of them.  On f16 pages 8 columns lie in both parts in one product.
constexpr int few_cols(bool f16) { return f16 ? 8 : 16; }
constexpr int step_keys(bool f16) { return f16 ? 32 : 16; }   // 8 KB of K and 8 KB of V, half of it on pages of 8 bits
template <typename CT>
constexpr bool is_q8 = std::is_same<CT, int8_t>::value;
template <typename CT>
constexpr bool f16_products = is_q8<CT> || std::is_same<CT, _Float16>::value;

struct AttnParams {
    const float * q;
    const void * pages;
    float * out;
    float * part_o;       // [rows * heads][n_parts][128]
    f2 * part_ml;         // [rows * heads][n_parts]: reference maximum (log2 units) and sum
    PagedSeqs seqs;
    int32_t n_heads, n_kv, group, n_pages, page_shift, layer;
    int32_t few_max;      // sequences of at most so many columns are of few columns
    int32_t tiles_many, tiles_few;   // upper bounds of both kinds of tiles
    int32_t splits_many, splits_few, steps_many, steps_few;   // key ranges of each kind, and their steps
    int32_t n_parts;      // ranges that the workspace holds of a (row, head): the more of the two
    float scale;
    const uint32_t * mask;   // trees: [rows][mask_words], bit i: the row sees its sequence's new token i
    int32_t mask_words;
};

__device__ inline uint32_t lo_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ inline uint32_t hi_pair(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ inline float column_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A tile of the batch: a sequence, its first column, and what its keys are.
struct Tile {
    const int32_t * table;
    int rows, row0, past;     // the sequence's new tokens, the first one's row and position
    int col0, n_cols;         // the tile's first column, the sequence's columns
    int cap, kend;            // positions of the table row; keys that the tile's last token sees
    int n_steps, step_lo, step_hi;   // steps of kend, and those of this split
    int split, n_splits;
};

// Block -> (KV head, split, tile); false: nothing to do.  Neighbouring blocks, which go to different XCDs, take different heads.
// Every lane counts one sequence's tiles, a prefix sum over the wave finds the sequence that holds the tile; what the tile
// needs is read along.  FEW: the sequences of 1 .. few_max columns, otherwise the longer ones.
template <int R, int KS, bool FEW, bool TREE>
__device__ inline bool find_tile(const AttnParams & p, int block, int lane, Tile & t, int & head) {
    const int n_tiles = FEW ? p.tiles_few : p.tiles_many, split_steps = FEW ? p.steps_few : p.steps_many;
    head = block % p.n_kv;
    const int rest = block / p.n_kv;
    t.split = rest / n_tiles;
    t.n_splits = FEW ? p.splits_few : p.splits_many;
    int tile = rest - t.split * n_tiles;
    for (int s0 = 0; s0 < p.seqs.n_seqs; s0 += kWave) {
        const int s = s0 + lane;
        int n = 0, rows = 0, start = 0, past = 0;
        if (s < p.seqs.n_seqs) {
            start = p.seqs.row_start[s];
            past = p.seqs.n_past[s];
            rows = rows_between(start, p.seqs.row_start[s + 1], p.seqs.n_rows);
            const bool few = rows * p.group <= p.few_max;
            if (rows > 0 && few == FEW) n = FEW ? 1 : (rows * p.group + R - 1) / R;
        }
        int sum = n;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const int o = __shfl_up(sum, d, kWave);
            if (lane >= d) sum += o;
        }
        const uint64_t holds = __ballot(sum > tile);
        if (holds != 0) {
            const int l = __ffsll(static_cast<unsigned long long>(holds)) - 1;
            const int count = __builtin_amdgcn_readlane(n, l), before = __builtin_amdgcn_readlane(sum, l) - count;
            t.table = p.seqs.tables + static_cast<int64_t>(s0 + l) * p.seqs.table_stride;
            t.rows = __builtin_amdgcn_readlane(rows, l);
            t.row0 = __builtin_amdgcn_readlane(start, l);
            t.past = bounded_past(__builtin_amdgcn_readlane(past, l));
            t.col0 = (count - 1 - (tile - before)) * R;               // the last tile has the most keys: first
            t.n_cols = t.rows * p.group;
            t.cap = p.seqs.table_stride << p.page_shift;
            t.kend = max(0, min(t.past + (TREE ? t.rows - 1 : (min(t.col0 + R, t.n_cols) - 1) / p.group), t.cap - 1) + 1);
            t.n_steps = (t.kend + KS - 1) / KS;
            t.step_lo = t.split * split_steps;
            t.step_hi = t.split == t.n_splits - 1 ? t.n_steps : min(t.n_steps, t.step_lo + split_steps);
            return t.split == 0 || t.step_lo < t.n_steps;               // the first split answers for rows without keys
        }
        tile -= __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    return false;
}

// A column: its output row (token and head; -1: none), the last position it sees and its q.
struct Column {
    int row, lim;
    const float * q;
    int mask;       // trees: its row's first word
};

template <bool TREE>
__device__ inline Column column_of(const AttnParams & p, const Tile & t, int head, int col) {
    const bool ok = col < t.n_cols;
    const int token = (ok ? col : t.n_cols - 1) / p.group;
    const int row = (t.row0 + token) * p.n_heads + head * p.group + (ok ? col - token * p.group : 0);
    return Column{ok ? row : -1, ok ? min(t.past + (TREE ? t.rows - 1 : token), t.cap - 1) : -1, p.q + static_cast<int64_t>(row) * kHeadDim,
                  TREE ? (t.row0 + token) * p.mask_words : 0};
}

// A table entry as the page of the 16 keys from j on, -1 for none.
__device__ inline int entry_page(const AttnParams & p, const Tile & t, int entry, int j) {
    return j < t.kend && entry >= 0 && entry < p.n_pages ? entry : -1;
}

// 32 bits of a row's mask from new token `first` on; cached positions (numbers below 0) are seen, those behind the mask are not.
__device__ inline uint32_t mask_window(const AttnParams & p, const uint32_t * words, int first) {
    const int w = first >> 5;
    const uint32_t lo = w < 0 ? ~0u : w < p.mask_words ? words[w] : 0u;
    const uint32_t hi = w + 1 < 0 ? ~0u : w + 1 < p.mask_words ? words[w + 1] : 0u;
    return __builtin_amdgcn_alignbit(hi, lo, first & 31);
}

__device__ inline const uint32_t * mask_row(const AttnParams & p, int row) {
    return p.mask + static_cast<int64_t>(row / p.n_heads) * p.mask_words;
}

// Whether any position that the row (token and head) sees lies on a page.
template <bool TREE>
__device__ inline bool sees_any(const AttnParams & p, const int32_t * table, int lim, int past, int row) {
    for (int j = 0; j <= (TREE ? min(lim, past - 1) : lim); j += 1 << p.page_shift) {
        if (page_of(table, p.seqs.table_stride, p.page_shift, p.n_pages, j) >= 0) return true;
    }
    if constexpr (TREE) {
        for (int j = max(past, 0); j <= lim; ++j) {
            if ((mask_window(p, mask_row(p, row), j - past) & 1u) && page_of(table, p.seqs.table_stride, p.page_shift, p.n_pages, j) >= 0) return true;
        }
    }
    return false;
}

// 1 / sum, 0 for a row that sees no key; a row whose visible scores are all -inf has sum 0 and is NaN by the formula.
template <bool TREE>
__device__ inline float inverse_sum(const AttnParams & p, const int32_t * table, int lim, int past, int row, float l) {
    if (l == 0.0f) return sees_any<TREE>(p, table, lim, past, row) ? NAN : 0.0f;
    return 1.0f / l;
}

// One column over the visible keys of steps step0, step0 + step_inc, .. < step1, in f32, key by key: lane holds dims
// 2 lane and 2 lane + 1.  m in log2 units.
template <typename CT, int KS, bool TREE>
__device__ inline void column_by_keys(const AttnParams & p, const int32_t * table, int head, int row, int lim, int past, int step0,
                                      int step1, int step_inc, int lane, float & m, float & l, f2 & o) {
    const f2 qv = *reinterpret_cast<const f2 *>(p.q + static_cast<int64_t>(row) * kHeadDim + 2 * lane);
    const float c = p.scale * kLog2e;
    const HeadRows<CT> rows(p.pages, p.layer, p.n_kv, p.n_pages, p.page_shift, head);
    m = -INFINITY;
    l = 0.0f;
    o = f2{0.0f, 0.0f};
    for (int st = step0; st < step1; st += step_inc) {
        for (int j = st * KS; j < st * KS + KS && j <= lim; ++j) {
            const int page = page_of(table, p.seqs.table_stride, p.page_shift, p.n_pages, j);
            if (page < 0) continue;
            if constexpr (TREE) {
                if (!(mask_window(p, mask_row(p, row), j - past) & 1u)) continue;
            }
            const int slot = j & ((1 << p.page_shift) - 1);
            const CT * k = rows.page(page) + slot * kHeadDim + 2 * lane;
            const CT * v = k + rows.v_elems;
            float ks = 1.0f, vs = 1.0f;
            if constexpr (is_q8<CT>) {
                ks = rows.scale(page)[slot];
                vs = rows.scale(page)[rows.v_elems / 4 + slot];
            }
            const float s = wave_sum_all(fmaf(qv[0], static_cast<float>(k[0]) * ks, qv[1] * (static_cast<float>(k[1]) * ks))) * c;
            const float mn = fmaxf(m, s);
            const float ref = mn == -INFINITY ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(s - ref);
            l = l * f + e;
            o[0] = o[0] * f + e * (static_cast<float>(v[0]) * vs);
            o[1] = o[1] * f + e * (static_cast<float>(v[1]) * vs);
            m = mn;
        }
    }
}

// A column's q in MFMA order: f16 pages dims 32 ks + 8 (l / 16) .. at [2 ks], pages of 8 bits dims 64 (ks / 2) + 16 (l / 16) +
// 8 (ks % 2) .. there, f32 pages dims 16 i + 4 (l / 16) .. at [i].  Columns that do not exist are zeros.
template <typename CT>
__device__ inline void load_q(const Column & col, int g4, f4 (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = *reinterpret_cast<const f4 *>(col.q + (is_q8<CT> ? (i >> 2) * 64 + g4 * 16 + (i & 3) * 4
                                                      : f16_products<CT> ? (i >> 1) * 32 + g4 * 8 + (i & 1) * 4 : i * 16 + g4 * 4));
        if (col.row < 0) x[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// A step of scores S^T = K Q^T from its 8 K operands.  Q: the two parts on f16 pages (the packed form has both in the first),
// the values themselves on f32 pages.
template <bool F16, bool PACK, int NB>
__device__ inline void scores_step(const u4 (&a)[8], const h8 (&qh)[NB][4], const h8 (&ql)[NB][4], const f4 (&x)[NB][8],
                                   f4 (&S)[NB][F16 ? 2 : 1]) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int kb = 0; kb < (F16 ? 2 : 1); ++kb) S[nb][kb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if constexpr (F16) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
            for (int part = 0; part < (PACK ? 1 : 2); ++part) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        S[nb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a[kb * 4 + ks]), part ? ql[nb][ks] : qh[nb][ks],
                                                                           S[nb][kb], 0, 0, 0);
                    }
                }
            }
        }
    } else {
        // two sums, so that a product does not wait for the one before it
        f4 T[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) T[nb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    f4 & to = e & 1 ? T[nb] : S[nb][0];
                    to = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f4, a[i])[e], x[nb][i][e], to, 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) S[nb][0] += T[nb];
    }
}

// -inf where a key lies behind the column's last position, on no page (bit kb of holes: the 16-key block kb) or outside its mask.
template <int NB, int KB, bool TREE>
__device__ inline void mask_step(const AttnParams & p, f4 (&S)[NB][KB], const int (&lim)[NB], const int (&mask)[NB], int past, int key0,
                                 int g4, int holes) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        uint32_t seen = ~0u;
        if constexpr (TREE) seen = mask_window(p, p.mask + mask[nb], key0 - past);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bool out = key0 + kb * 16 + g4 * 4 + i > lim[nb] || ((holes >> kb) & 1);
                if constexpr (TREE) out = out || !((seen >> (kb * 16 + g4 * 4 + i)) & 1u);
                if (out) S[nb][kb][i] = -INFINITY;
            }
        }
    }
}

// V^T operand db of a step's f16 rows: dims 8 r + db, two keys per register.
__device__ inline u4 transposed(const u4 (&v)[8], int db) {
    u4 a;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        a[w] = db & 1 ? hi_pair(v[2 * w][db >> 1], v[2 * w + 1][db >> 1]) : lo_pair(v[2 * w][db >> 1], v[2 * w + 1][db >> 1]);
    }
    return a;
}

// 8 bits as f16: one instruction per value, which takes its byte and leaves the other half of the register.  The s_nop behind 16
// of them is the wait that a reader of a half-written register needs.
__device__ inline void f16_words(u4 raw, u4 & lo, u4 & hi) {             // 16 bytes in order
    uint32_t o[8];
    asm("v_cvt_f16_i16_sdwa %0, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
        "v_cvt_f16_i16_sdwa %1, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
        "v_cvt_f16_i16_sdwa %2, sext(%9) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
        "v_cvt_f16_i16_sdwa %3, sext(%9) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
        "v_cvt_f16_i16_sdwa %4, sext(%10) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
        "v_cvt_f16_i16_sdwa %5, sext(%10) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
        "v_cvt_f16_i16_sdwa %6, sext(%11) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
        "v_cvt_f16_i16_sdwa %7, sext(%11) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
        "v_cvt_f16_i16_sdwa %0, sext(%8) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_1\n\t"
        "v_cvt_f16_i16_sdwa %1, sext(%8) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_3\n\t"
        "v_cvt_f16_i16_sdwa %2, sext(%9) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_1\n\t"
        "v_cvt_f16_i16_sdwa %3, sext(%9) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_3\n\t"
        "v_cvt_f16_i16_sdwa %4, sext(%10) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_1\n\t"
        "v_cvt_f16_i16_sdwa %5, sext(%10) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_3\n\t"
        "v_cvt_f16_i16_sdwa %6, sext(%11) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_1\n\t"
        "v_cvt_f16_i16_sdwa %7, sext(%11) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_3\n\t"
        "s_nop 0"
        : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3]), "=&v"(o[4]), "=&v"(o[5]), "=&v"(o[6]), "=&v"(o[7])
        : "v"(raw[0]), "v"(raw[1]), "v"(raw[2]), "v"(raw[3]));
    lo = u4{o[0], o[1], o[2], o[3]};
    hi = u4{o[4], o[5], o[6], o[7]};
}

// K operands 4 kb .. 4 kb + 3 of a step from the lane's 2 x 16 bytes of 16-key block kb.
__device__ inline void k_operands(const u4 (&raw)[4], u4 (&a)[8]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) f16_words(raw[r], a[2 * r], a[2 * r + 1]);
}

// V^T operands 4 h + 2 D and 4 h + 2 D + 1 of a step's rows of 8 bits, 8 dims per lane and key: two keys' values per word.
template <int D>
__device__ inline void v_operands(const u2 (&raw)[8], int h, u4 & even, u4 & odd) {
    uint32_t o[8];
    if constexpr (D == 0) {
        asm("v_cvt_f16_i16_sdwa %0, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
            "v_cvt_f16_i16_sdwa %4, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1\n\t"
            "v_cvt_f16_i16_sdwa %1, sext(%10) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
            "v_cvt_f16_i16_sdwa %5, sext(%10) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1\n\t"
            "v_cvt_f16_i16_sdwa %2, sext(%12) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
            "v_cvt_f16_i16_sdwa %6, sext(%12) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1\n\t"
            "v_cvt_f16_i16_sdwa %3, sext(%14) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0\n\t"
            "v_cvt_f16_i16_sdwa %7, sext(%14) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1\n\t"
            "v_cvt_f16_i16_sdwa %0, sext(%9) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_0\n\t"
            "v_cvt_f16_i16_sdwa %4, sext(%9) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_1\n\t"
            "v_cvt_f16_i16_sdwa %1, sext(%11) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_0\n\t"
            "v_cvt_f16_i16_sdwa %5, sext(%11) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_1\n\t"
            "v_cvt_f16_i16_sdwa %2, sext(%13) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_0\n\t"
            "v_cvt_f16_i16_sdwa %6, sext(%13) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_1\n\t"
            "v_cvt_f16_i16_sdwa %3, sext(%15) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_0\n\t"
            "v_cvt_f16_i16_sdwa %7, sext(%15) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_1\n\t"
            "s_nop 0"
            : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3]), "=&v"(o[4]), "=&v"(o[5]), "=&v"(o[6]), "=&v"(o[7])
            : "v"(raw[0][h]), "v"(raw[1][h]), "v"(raw[2][h]), "v"(raw[3][h]), "v"(raw[4][h]), "v"(raw[5][h]), "v"(raw[6][h]), "v"(raw[7][h]));
    } else {
        asm("v_cvt_f16_i16_sdwa %0, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
            "v_cvt_f16_i16_sdwa %4, sext(%8) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3\n\t"
            "v_cvt_f16_i16_sdwa %1, sext(%10) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
            "v_cvt_f16_i16_sdwa %5, sext(%10) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3\n\t"
            "v_cvt_f16_i16_sdwa %2, sext(%12) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
            "v_cvt_f16_i16_sdwa %6, sext(%12) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3\n\t"
            "v_cvt_f16_i16_sdwa %3, sext(%14) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
            "v_cvt_f16_i16_sdwa %7, sext(%14) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3\n\t"
            "v_cvt_f16_i16_sdwa %0, sext(%9) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_2\n\t"
            "v_cvt_f16_i16_sdwa %4, sext(%9) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_3\n\t"
            "v_cvt_f16_i16_sdwa %1, sext(%11) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_2\n\t"
            "v_cvt_f16_i16_sdwa %5, sext(%11) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_3\n\t"
            "v_cvt_f16_i16_sdwa %2, sext(%13) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_2\n\t"
            "v_cvt_f16_i16_sdwa %6, sext(%13) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_3\n\t"
            "v_cvt_f16_i16_sdwa %3, sext(%15) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_2\n\t"
            "v_cvt_f16_i16_sdwa %7, sext(%15) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_3\n\t"
            "s_nop 0"
            : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3]), "=&v"(o[4]), "=&v"(o[5]), "=&v"(o[6]), "=&v"(o[7])
            : "v"(raw[0][h]), "v"(raw[1][h]), "v"(raw[2][h]), "v"(raw[3][h]), "v"(raw[4][h]), "v"(raw[5][h]), "v"(raw[6][h]), "v"(raw[7][h]));
    }
    even = u4{o[0], o[1], o[2], o[3]};
    odd = u4{o[4], o[5], o[6], o[7]};
}

// Element offset of operand f of a step inside its 16-key block, and that block.  K on f16 pages: key l % 16, dims as q's.  V there:
// key 16 (f / 4) + 4 (l / 16) + f % 4, dims 8 (l % 16) ..; on f32 pages key 4 (l / 16) + f / 2, dims 8 (l % 16) + 4 (f % 2) ...
__device__ inline int k_offset(int f, int c16, int g4) { return c16 * kHeadDim + (f & 3) * 32 + g4 * 8; }
template <bool F16>
__device__ inline int v_offset(int f, int c16, int g4) {
    return F16 ? (g4 * 4 + (f & 3)) * kHeadDim + c16 * 8 : (g4 * 4 + (f >> 1)) * kHeadDim + c16 * 8 + (f & 1) * 4;
}
template <bool F16>
__device__ inline int v_key(int f, int g4) { return F16 ? (f >> 2) * 16 + g4 * 4 + (f & 3) : g4 * 4 + (f >> 1); }

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

// The same on pages of 8 bits, where the keys' V scales go into the probabilities, which are split into f16 parts behind that.  So that
// these keep their bits whatever the scales are, the column's reference (log2 units) follows the largest product that the
// column has: w = exp2(s - m) scale <= 2^14, and a key that it does not see, or hardly, moves nothing, however large its row.
// Probabilities alone are in m, too, f32 as their sum is, and up to 2^95: scales below 2^kLeastScale, and 0, count as that.  What a column
// sees of rows so small (but not 0) it computes again key by key (small).
// Scales of one size, the common case, are bounded per lane by the largest of its 8: at most 6 bits more than needed.  (1024 tokens behind
// 2889 positions 72.6 us; 78 where all steps have scales up to 2^10 apart, 32 streams 32.0 / 32.9.)  m is whole, so that sum and
// accumulators follow it without rounding, over any distance.
constexpr float kLeastScale = -80.0f;
constexpr float kNearScales = 0x1p-6f, kSmallScale = 0x1p-78f;
__device__ inline float log2_near(float x) {                          // up to 0.09 below; 128 and more of what is not finite
    return fmaf(static_cast<float>(__float_as_uint(x)), 0x1p-23f, -127.0f);
}

// The scales of rows that no column sees (keys from `keys` on, blocks of holes): any finite one will do, as their probability is 0; one of the
// lane's others keeps the step to scales of one size (one token behind 156 positions 6.50 us, with zeros 6.70; attn_wide, whose
// registers it costs, has zeros: sixteen trees of up to 41 nodes 34.7, so 35.7).
__device__ inline void neutral_scales(f4 (&vs)[2], int keys, int holes, int g4) {
    float other = 0.0f;
#pragma unroll
    for (int f = 0; f < 8; ++f) {
        const bool none = v_key<true>(f, g4) >= keys || ((holes >> (f >> 2)) & 1);
        other = fmaxf(other, none ? 0.0f : vs[f >> 2][f & 3]);
    }
    if (!(other > 0.0f && other < INFINITY)) other = 1.0f;
#pragma unroll
    for (int f = 0; f < 8; ++f) {
        if (v_key<true>(f, g4) >= keys || ((holes >> (f >> 2)) & 1)) vs[f >> 2][f & 3] = other;
    }
}

template <int NB>
__device__ inline void weighted_step(const f4 (&S)[NB][2], const f4 (&vs)[2], const float (&c)[NB], float (&m)[NB], float (&l)[NB],
                                     f4 (&O)[NB][8], float (&pr)[NB][2][4], bool & small) {
    float most = 0.0f, least = INFINITY, t[NB];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            most = fmaxf(most, vs[kb][i]);
            least = fminf(least, vs[kb][i]);
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) t[nb] = -INFINITY;
    if (!__any(!(least >= fmaxf(most * kNearScales, kSmallScale)))) {
        const float size = log2_near(most);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                for (int i = 0; i < 4; ++i) t[nb] = fmaxf(t[nb], S[nb][kb][i]);
            }
            t[nb] = fmaf(t[nb], c[nb], size);
        }
    } else {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = fabsf(vs[kb][i]), size = fmaxf(log2_near(x), kLeastScale);
                bool seen = false;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    t[nb] = fmaxf(t[nb], fmaf(S[nb][kb][i], c[nb], size));
                    seen = seen || S[nb][kb][i] > -INFINITY;
                }
                small = small || (seen && x > 0.0f && x < kSmallScale);
            }
        }
    }
    float mn[NB];
    bool up[NB], any = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        mn[nb] = fmaxf(m[nb], column_max(t[nb]));
        up[nb] = mn[nb] - m[nb] > kLazyLog2;             // -inf to finite: yes; -inf to -inf: NaN, no
        any = any || up[nb];
    }
    if (__any(any)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float to = rintf(mn[nb]);
            const int by = up[nb] ? static_cast<int>(fmaxf(m[nb] - to, -1000.0f)) : 0;
#pragma unroll
            for (int db = 0; db < 8; ++db) {
#pragma unroll
                for (int i = 0; i < 4; ++i) O[nb][db][i] = ldexpf(O[nb][db][i], by);
            }
            l[nb] = ldexpf(l[nb], by);
            if (up[nb]) m[nb] = to;
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const float mc = m[nb] == -INFINITY ? INFINITY : m[nb] - kShiftLog2;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(S[nb][kb][i], c[nb], -mc));
                l[nb] += e;
                pr[nb][kb][i] = e * vs[kb][i];
                // the product as it is rounded here: one that a conversion to f16 takes in unrounded (v_fma_mix) is now and then
                // another f16 than the one whose rest is the second part
                asm("" : "+v"(pr[nb][kb][i]));
            }
        }
    }
}

// Probabilities as two f16 parts in the order of the PV product.  The rest v - hi is one instruction that takes hi as f16
// (v_fma_mix_f32; the factor is hidden, or the compiler makes a conversion and a difference of it).
__device__ inline void split_p(const float (&pr)[2][4], h8 & hi, h8 & lo) {
    float minus = -1.0f;
    asm("" : "+s"(minus));
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const f2 v = {pr[e >> 2][e & 3], pr[e >> 2][(e & 3) + 1]};
        const h2 h = __builtin_convertvector(v, h2);
        const f2 rest = {fmaf(static_cast<float>(h[0]), minus, v[0]), fmaf(static_cast<float>(h[1]), minus, v[1])};
        const h2 r = __builtin_convertvector(rest, h2);
        hi[e] = h[0];
        hi[e + 1] = h[1];
        lo[e] = r[0];
        lo[e + 1] = r[1];
    }
}

// 4 values of a column from dim on: the output, or the part of this split (lead: this lane also stores the part's weights).
template <bool TREE>
__device__ inline void store_column(const AttnParams & p, const Tile & t, int row, int lim, int dim, f4 v, float mc, float l, bool lead) {
    if (t.n_splits == 1) {
        *reinterpret_cast<f4 *>(p.out + static_cast<int64_t>(row) * kHeadDim + dim) = v * inverse_sum<TREE>(p, t.table, lim, t.past, row, l);
    } else {
        const int64_t at = static_cast<int64_t>(row) * p.n_parts + t.split;
        *reinterpret_cast<f4 *>(p.part_o + at * kHeadDim + dim) = v;
        if (lead) p.part_ml[at] = f2{mc, l};
    }
}

// The end of a wave's steps: the column's sum over its 4 lanes, its reference in log2 units, and the columns of each block
// whose values are not all finite, or flagged (again).  WEIGHTED: m is weighted_step's, and the sums, which may be of any size, are brought to 1/2 .. 1,
// so that the reference says what they weigh beside other waves' and ranges'.
template <int NB, bool PACK, bool WEIGHTED>
__device__ inline void close_columns(const int (&orow)[NB], const float (&c)[NB], const float (&m)[NB], float (&l)[NB], f4 (&O)[NB][8],
                                     float (&mc)[NB], uint32_t (&redo)[NB], bool again) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        l[nb] = column_sum(l[nb]);
        mc[nb] = m[nb] == -INFINITY ? -INFINITY : WEIGHTED ? m[nb] - kShiftLog2 : fmaf(m[nb], c[nb], -kShiftLog2);
        int ex = 0;
        if constexpr (WEIGHTED) {
            ex = __builtin_amdgcn_frexp_expf(l[nb]);                  // 0 of 0 and of what is not finite
            l[nb] = ldexpf(l[nb], -ex);
            mc[nb] += static_cast<float>(ex);
        }
        // 0 x is 0 unless x is not finite, and a sum of such products is then NaN
        float zero = 0.0f * l[nb];
#pragma unroll
        for (int db = 0; db < 8; ++db) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (PACK) O[nb][db][i] += row_ror8(O[nb][db][i]);
                if constexpr (WEIGHTED) O[nb][db][i] = ldexpf(O[nb][db][i], -ex);
                zero = fmaf(0.0f, O[nb][db][i], zero);
            }
        }
        const uint64_t bad = __ballot((!(zero == 0.0f) || m[nb] == INFINITY || again) && orow[nb] >= 0);
        redo[nb] = static_cast<uint32_t>(bad | (bad >> 16) | (bad >> 32) | (bad >> 48)) & (PACK ? 0xffu : 0xffffu);
    }
}

// The flagged columns of a block, key by key; their values are stored at once.
template <typename CT, int KS>
__device__ inline void redo_columns(const AttnParams & p, const Tile & t, int head, int lane, int lim, int orow, uint32_t redo) {
    for (uint32_t left = redo; left != 0; left &= left - 1) {
        const int col = __ffs(left) - 1;
        const int row = __builtin_amdgcn_readlane(orow, col), lm = __builtin_amdgcn_readlane(lim, col);
        float cm, cl;
        f2 co;
        column_by_keys<CT, KS, false>(p, t.table, head, row, lm, t.past, t.step_lo, t.step_hi, 1, lane, cm, cl, co);
        const f2 nx = f2{__shfl_down(co[0], 1, kWave), __shfl_down(co[1], 1, kWave)};
        if ((lane & 1) == 0) store_column<false>(p, t, row, lm, 2 * lane, f4{co[0], co[1], nx[0], nx[1]}, cm, cl, lane == 0);
    }
}

// Up to 16 columns (FEW on f16 pages: 8, in both parts), whose keys the waves take in turn, step by step, each its own K and V, with no
// barrier between the steps: a decode step is the stream of K and V, and the next step's loads are under way behind the
// products.  The waves' results are merged in LDS.  32 decode steps behind 156 to 3914 positions on 8 bits (137 MB) 30.8 us, 4.5 TB/s of the
// 5.1 that a copy reaches.
constexpr int kRowsStride = kHeadDim + 4;
constexpr int rows_cols(bool f16, bool few) { return f16 && few ? 8 : 16; }
constexpr size_t rows_lds(bool f16, bool few, int waves = kWaves) { return waves * rows_cols(f16, few) * (kRowsStride + 2) * 4 + 2 * rows_cols(f16, few) * 4; }

// A sequence that is one tile on f16 pages reads its K and V once, whole lines at a time: past the caches (ONCE).  32 sequences of
// 3914 positions 84 instead of 94 us, of 157 to 3914 55.7 instead of 57.3 (8 bits: V alone 30.4 us, both 31.4, neither 35.3).  That is
// for sequences with pages of their own; what
// forked ones share is read once by each of them, and finds less of it in the caches: 32 beams behind 3913 shared positions 46.8
// us, cached 42.6, behind 1000 19.2 / 18.5, eight behind 3913 22.3 / 21.1.  Nothing tells the two apart before the tables are read.  A row
// of f32 pages is taken by halves of its lines, and longer chunks read it again: 129 instead of 111 us, and 50 instead of 40 at eight of 64 tokens.
template <bool ONCE, typename VT>
__device__ inline VT load_row(const void * at) {
    if constexpr (ONCE) return __builtin_nontemporal_load(static_cast<const VT *>(at));
    else return *static_cast<const VT *>(at);
}

// A step of K in LDS, a wave's own.  A load instruction brings whole rows straight into LDS, a kilobyte in the order of its lanes, 16
// bytes each; which of its row's 16 bytes a lane takes depends on the row, so that the 16 rows of an operand are read from different
// banks.  (A lane that loads its own operand takes 16 bytes of a row per instruction, and the 15 beside it as many other rows: four
// times the cache accesses, and registers for all of it.  Sixteen trees of up to 41 nodes 43 us so, 37 through LDS, decode steps on
// 8 bits 35.7 / 30.4, one tree of 64 10.7 / 9.0.)
template <typename CT, bool ONCE = false>
struct KStep {
    static constexpr int kRow = kHeadDim * sizeof(CT), kInRow = kRow / 16, kAtOnce = kWave / kInRow, kPerBlock = 16 / kAtOnce;
    static constexpr int kBlocks = step_keys(f16_products<CT>) / 16, kBytes = kBlocks * 16 * kRow;
    char * lds;
    uint32_t lane_at[kPerBlock];
    static __device__ inline int turn(int key) { return is_q8<CT> ? (key >> 1) & 7 : key & 15; }
    __device__ inline KStep(char * to, int lane) : lds(to) {
#pragma unroll
        for (int f = 0; f < kPerBlock; ++f) {
            const int key = f * kAtOnce + lane / kInRow;
            lane_at[f] = key * kRow + ((lane % kInRow) ^ turn(key)) * 16;
        }
    }
    // at: the step's 16-key blocks.  Buffer loads, as the compiler counts them like any other (after global loads into LDS it waits for all).
    __device__ inline void load([[maybe_unused]] const CT * const * at) const {
#ifdef __HIP_DEVICE_COMPILE__                              // the host has no type for the buffer
#pragma unroll
        for (int f = 0; f < kBlocks * kPerBlock; ++f) {
            const auto block = __builtin_amdgcn_make_buffer_rsrc(const_cast<CT *>(at[f / kPerBlock]), 0, 16 * kRow, 0x00027000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(block, (__attribute__((address_space(3))) void *)(lds + f * 1024), 16, lane_at[f % kPerBlock], 0, 0,
                                                     ONCE ? 2 : 0);
        }
#endif
    }
    // Behind K's loads: none of V's, which arrived() counts, is moved ahead of them.
    static __device__ inline void issued() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0x81);              // what is no access of memory, or one of LDS, may pass
    }
    // Before a step's chunks are read: of the loads behind those of K there are V's 8.
    static __device__ inline void arrived() { asm volatile("s_waitcnt vmcnt(8)" ::: "memory"); }
    // Before the next step is loaded: this one has been read.
    static __device__ inline void read() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xc07f);                // lgkmcnt(0)
    }
    __device__ inline u4 chunk(int kb, int c16, int chunk) const {
        return *reinterpret_cast<const u4 *>(lds + kb * 16 * kRow + c16 * kRow + (chunk ^ turn(c16)) * 16);
    }
};

// LDS of attn_rows: its waves' K, then their results.
template <typename CT>
constexpr size_t rows_bytes(bool few, int waves = kWaves) { return std::max<size_t>(rows_lds(f16_products<CT>, few, waves), waves * KStep<CT>::kBytes); }

// The table of a tile, for scalar loads, which the loads into LDS would rule out for memory that might be written.
__device__ inline const __attribute__((address_space(4))) int32_t * scalar_table(const Tile & t) {
    return reinterpret_cast<const __attribute__((address_space(4))) int32_t *>(reinterpret_cast<uintptr_t>(t.table));
}

// The W waves' results of R columns, merged in LDS and stored; what is to be computed again (redo) is, key by key.
template <typename CT, int R, bool PACK, bool TREE, int W>
__device__ inline void merge_waves(const AttnParams & p, const Tile & t, int head, char * lds, int wave, int lane, int orow, int lim, float mc,
                                   float l, const f4 (&O)[8], uint32_t redo) {
    constexpr int KS = step_keys(f16_products<CT>);
    const int c16 = lane & 15, g4 = lane >> 4;
    float * so = reinterpret_cast<float *>(lds);
    float * sm = so + W * R * kRowsStride;
    float * sl = sm + W * R;
    int * srow = reinterpret_cast<int *>(sl + W * R);
    int * slim = srow + R;
    const int base = wave * R;
    if (!PACK || c16 < 8) {
        float * to = so + (base + c16) * kRowsStride + g4 * 32;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                *reinterpret_cast<f4 *>(to + i * 8 + h * 4) = f4{O[4 * h][i], O[4 * h + 1][i], O[4 * h + 2][i], O[4 * h + 3][i]};
            }
        }
        if (g4 == 0) {
            sm[base + c16] = mc;
            sl[base + c16] = l;
            if (wave == 0) {
                srow[c16] = orow;
                slim[c16] = lim;
            }
        }
    }
    for (uint32_t left = redo; left != 0; left &= left - 1) {
        const int cc = __ffs(left) - 1;
        const int row = __builtin_amdgcn_readlane(orow, cc), lm = __builtin_amdgcn_readlane(lim, cc);
        float cm, cl;
        f2 co;
        column_by_keys<CT, KS, TREE>(p, t.table, head, row, lm, t.past, t.step_lo + wave, t.step_hi, W, lane, cm, cl, co);
        // after this wave's own stores above: one wave's LDS accesses stay in order
        __builtin_amdgcn_wave_barrier();
        *reinterpret_cast<f2 *>(so + (base + cc) * kRowsStride + 2 * lane) = co;
        if (lane == 0) {
            sm[base + cc] = cm;
            sl[base + cc] = cl;
        }
    }
    __syncthreads();
#pragma unroll
    for (int idx = threadIdx.x; idx < R * (kHeadDim / 4); idx += W * kWave) {
        const int cc = idx / (kHeadDim / 4), dim = (idx % (kHeadDim / 4)) * 4;
        const int row = srow[cc];
        if (row < 0) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w * R + cc]);
        float ls = 0.0f;
        f4 o = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float mw = sm[w * R + cc];
            const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - M);
            ls += sl[w * R + cc] * f;
            o += *reinterpret_cast<const f4 *>(so + (w * R + cc) * kRowsStride + dim) * f;
        }
        store_column<TREE>(p, t, row, slim[cc], dim, o, M, ls, dim == 0);
    }
}

template <typename CT, bool FEW, bool TREE, int W>
__device__ inline void attn_rows(const AttnParams & p, int block, char * lds) {
    constexpr bool F16 = f16_products<CT>, Q8 = is_q8<CT>, PACK = FEW && F16;
    constexpr int KS = step_keys(F16), KB = KS / 16, R = rows_cols(F16, FEW), NB = 1;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    Tile t;
    int head;
    if (!find_tile<R, KS, FEW, TREE>(p, block, lane, t, head)) return;    // uniform for the workgroup
    const Column col = column_of<TREE>(p, t, head, t.col0 + (PACK ? c16 & 7 : c16));
    f4 x[NB][8];
    load_q<CT>(col, g4, x[0]);

    const HeadRows<CT> rows(p.pages, p.layer, p.n_kv, p.n_pages, p.page_shift, head);
    const int in_page = (1 << p.page_shift) - 1, last_entry = p.seqs.table_stride - 1;
    const auto * table = scalar_table(t);
    auto entries_of = [&](int st, int (&out)[KB]) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) out[kb] = table[min((st * KS + kb * 16) >> p.page_shift, last_entry)];
    };
    // a lane's rows of a step of V; 8 bits: 8 bytes per key, and the scales of its 4 keys per 16-key block, K's and V's
    const KStep<CT, PACK && !Q8> k_step(lds + wave * KStep<CT>::kBytes, lane);
    u4 rv[Q8 ? 1 : 8];
    u2 rv8[8];
    f4 ks[KB], vs_next[KB];
    int pg[KB], pg_next[KB], entry[KB];
    const CT * at[KB];
    const char * scales[KB];
    // 8 bits: a lane's place in a 16-key block's V and scales, so that addresses are a uniform base and these
    const uint32_t v_lane = g4 * 4 * kHeadDim + c16 * 8, scale_lane = g4 * 16;
    // a block on no page reads page 0, which there always is, and is masked
    auto place = [&](int st) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            pg_next[kb] = entry_page(p, t, entry[kb], st * KS + kb * 16);
            at[kb] = rows.page(max(pg_next[kb], 0)) + ((st * KS + kb * 16) & in_page) * kHeadDim;
            if constexpr (Q8) scales[kb] = reinterpret_cast<const char *>(rows.scale(max(pg_next[kb], 0)) + ((st * KS + kb * 16) & in_page));
        }
    };
    auto load_k = [&]() {
        k_step.load(at);
        if constexpr (Q8) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                ks[kb] = *reinterpret_cast<const f4 *>(scales[kb] + scale_lane);
                vs_next[kb] = *reinterpret_cast<const f4 *>(scales[kb] + rows.v_elems + scale_lane);
            }
        }
        KStep<CT>::issued();
    };
    auto load_v = [&]() {
        if constexpr (Q8) {
#pragma unroll
            for (int f = 0; f < 8; ++f) rv8[f] = load_row<PACK, u2>(at[f >> 2] + rows.v_elems + v_lane + (f & 3) * kHeadDim);
        } else {
#pragma unroll
            for (int f = 0; f < 8; ++f) rv[f] = load_row<PACK, u4>(at[F16 ? f >> 2 : 0] + rows.v_elems + v_offset<F16>(f, c16, g4));
        }
    };
    int st = t.step_lo + wave;
    if (st < t.step_hi) {
        entries_of(st, entry);
        place(st);
        load_k();
        load_v();
        entries_of(st + W, entry);
    }

    float c[NB];
    h8 qh[NB][4], ql[NB][4];
    if constexpr (F16) {
        split_q(x[0], p.scale, c[0], qh[0], ql[0]);
        if constexpr (PACK) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) qh[0][ks] = c16 < 8 ? qh[0][ks] : ql[0][ks];
        }
    } else {
        c[0] = p.scale * kLog2e;
    }
    const int lim[NB] = {col.lim}, orow[NB] = {col.row}, mask[NB] = {col.mask};
    // steps that every column sees whole
    const int full = TREE ? max(0, min(t.past, t.cap)) / KS : max(0, min(t.past + t.col0 / p.group, t.cap - 1) + 1) / KS;
    [[maybe_unused]] bool small = false;
    float m[NB] = {-INFINITY}, l[NB] = {0.0f};
    f4 O[NB][8];
#pragma unroll
    for (int db = 0; db < 8; ++db) O[0][db] = f4{0.0f, 0.0f, 0.0f, 0.0f};

    // A step; more: the next one's rows are loaded on the way.  Loads under a condition would make every wait one for all loads.
    auto step = [&](auto more) {
        int holes = 0;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            pg[kb] = pg_next[kb];
            holes |= pg[kb] < 0 ? 1 << kb : 0;
        }
        f4 S[NB][KB], key_scale[KB], vs[KB];
        u4 a[8];
        k_step.arrived();
        if constexpr (Q8) {
            u4 raw[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) raw[f] = k_step.chunk(f >> 1, c16, (f & 1) * 4 + g4);
            k_operands(raw, a);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) key_scale[kb] = ks[kb], vs[kb] = vs_next[kb];
        } else {
#pragma unroll
            for (int f = 0; f < 8; ++f) a[f] = F16 ? k_step.chunk(f >> 2, c16, (f & 3) * 4 + g4) : k_step.chunk(0, c16, f * 4 + g4);
        }
        scores_step<F16, PACK, NB>(a, qh, ql, x, S);
        if constexpr (more.value) {
            place(st + W);
            k_step.read();
            load_k();
        }
        if constexpr (PACK) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
                for (int i = 0; i < 4; ++i) S[0][kb][i] += row_ror8(S[0][kb][i]);
            }
        }
        if constexpr (Q8) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) S[0][kb] *= key_scale[kb];
        }
        if (st >= full || holes != 0) mask_step<NB, KB, TREE>(p, S, lim, mask, t.past, st * KS, g4, holes);
        // rows of keys that no column sees, and of no page, are whatever memory holds: not even 0 times that
        if (st * KS + KS > t.kend || holes != 0) {
            if constexpr (Q8) {
                neutral_scales(vs, t.kend - st * KS, holes, g4);
            } else {
#pragma unroll
                for (int f = 0; f < 8; ++f) {
                    if (st * KS + v_key<F16>(f, g4) >= t.kend || pg[F16 ? f >> 2 : 0] < 0) rv[f] = u4{0, 0, 0, 0};
                }
            }
        }
        float pr[NB][KB][4];
        if constexpr (Q8) {
            weighted_step<NB>(S, vs, c, m, l, O, pr, small);
        } else {
            softmax_step<NB, KB>(S, c, m, l, O, pr);
        }
        if constexpr (F16) {
            h8 ph, pl;
            split_p(pr[0], ph, pl);
            if constexpr (PACK) ph = c16 < 8 ? ph : pl;
            u4 vt[2];
#pragma unroll
            for (int db = 0; db < 8; ++db) {
                if constexpr (!Q8) vt[db & 1] = transposed(rv, db);
                else if (db % 4 == 0) v_operands<0>(rv8, db >> 2, vt[0], vt[1]);
                else if (db % 4 == 2) v_operands<1>(rv8, db >> 2, vt[0], vt[1]);
                const h8 a = __builtin_bit_cast(h8, vt[db & 1]);
                O[0][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, O[0][db], 0, 0, 0);
                if constexpr (!PACK) O[0][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, O[0][db], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int f = 0; f < 8; ++f) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    O[0][(f & 1) * 4 + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f4, rv[f])[e], pr[0][0][f >> 1],
                                                                                 O[0][(f & 1) * 4 + e], 0, 0, 0);
                }
            }
        }
        if constexpr (more.value) {
            load_v();
            entries_of(st + 2 * W, entry);
        }
    };
    for (; st + W < t.step_hi; st += W) step(std::true_type{});
    if (st < t.step_hi) step(std::false_type{});

    float mc[NB];
    uint32_t redo[NB];
    close_columns<NB, PACK, Q8>(orow, c, m, l, O, mc, redo, small);
    __syncthreads();                                                      // every wave has read its K
    merge_waves<CT, R, PACK, TREE, W>(p, t, head, lds, wave, lane, col.row, col.lim, mc[0], l[0], O[0], redo[0]);
}

// 32 columns whose keys the waves take in turn, as in attn_rows, but with their q in LDS, where the waves read the operands of
// each step: a wave's registers hold the accumulators, and one read of K and V, and on 8 bits one conversion, serves all columns.  1024
// tokens behind 2889 positions on 8 bits (57 GF with both parts) 73 us, 780 TF/s where a large f16 product reaches 1147: two waves per
// SIMD, whose 330 other instructions per 64 products do not all find the matrix unit busy.  Three waves (168 registers, q and K read
// in smaller pieces) 77; more columns do not fit the registers.
constexpr int kWideBlocks = 2;
constexpr int kWideCols = 16 * kWideBlocks;
constexpr size_t kWideQ = kWideBlocks * 8 * kWave * 16;               // two parts of 4 operands per 16 columns
constexpr size_t kWideK = kWideQ + 1024;                              // behind q and its units: a step of K per wave
template <typename CT>
constexpr size_t wide_lds(int waves) { return std::max<size_t>(kWideK + waves * KStep<CT>::kBytes, rows_lds(true, false, waves)); }

template <typename CT, bool TREE, int W>
__device__ inline void attn_wide(const AttnParams & p, int block, char * lds) {
    constexpr bool Q8 = is_q8<CT>;
    constexpr int KS = step_keys(true), KB = KS / 16, NB = kWideBlocks;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    Tile t;
    int head;
    if (!find_tile<kWideCols, KS, false, TREE>(p, block, lane, t, head)) return;   // uniform for the workgroup

    const HeadRows<CT> rows(p.pages, p.layer, p.n_kv, p.n_pages, p.page_shift, head);
    const int in_page = (1 << p.page_shift) - 1, last_entry = p.seqs.table_stride - 1;
    const auto * table = scalar_table(t);
    auto entries_of = [&](int st, int (&out)[KB]) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) out[kb] = table[min((st * KS + kb * 16) >> p.page_shift, last_entry)];
    };
    u4 rv[Q8 ? 1 : 8];
    u2 rv8[8];
    f4 ks[KB], vs_next[KB];
    int pg[KB], pg_next[KB], entry[KB];
    const CT * at[KB];
    const char * scales[KB];
    const KStep<CT> k_step(lds + kWideK + wave * KStep<CT>::kBytes, lane);
    // 8 bits: a lane's place in a 16-key block's V and scales, so that addresses are a uniform base and these
    const uint32_t v_lane = g4 * 4 * kHeadDim + c16 * 8, scale_lane = g4 * 16;
    // a block on no page reads page 0, which there always is, and is masked
    auto place = [&](int st) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            pg_next[kb] = entry_page(p, t, entry[kb], st * KS + kb * 16);
            at[kb] = rows.page(max(pg_next[kb], 0)) + ((st * KS + kb * 16) & in_page) * kHeadDim;
            if constexpr (Q8) scales[kb] = reinterpret_cast<const char *>(rows.scale(max(pg_next[kb], 0)) + ((st * KS + kb * 16) & in_page));
        }
    };
    auto load_k = [&]() {
        k_step.load(at);
        if constexpr (Q8) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                ks[kb] = *reinterpret_cast<const f4 *>(scales[kb] + scale_lane);
                vs_next[kb] = *reinterpret_cast<const f4 *>(scales[kb] + rows.v_elems + scale_lane);
            }
        }
        KStep<CT>::issued();
    };
    auto load_v = [&]() {
        if constexpr (Q8) {
#pragma unroll
            for (int f = 0; f < 8; ++f) rv8[f] = *reinterpret_cast<const u2 *>(at[f >> 2] + rows.v_elems + v_lane + (f & 3) * kHeadDim);
        } else {
#pragma unroll
            for (int f = 0; f < 8; ++f) rv[f] = *reinterpret_cast<const u4 *>(at[f >> 2] + rows.v_elems + v_offset<true>(f, c16, g4));
        }
    };
    int st = t.step_lo + wave;
    if (st < t.step_hi) {
        entries_of(st, entry);
        place(st);
        load_k();
        load_v();
        entries_of(st + W, entry);
    }

    int lim[NB], orow[NB], mask[NB];
    float c[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const Column col = column_of<TREE>(p, t, head, t.col0 + nb * 16 + c16);
        lim[nb] = col.lim;
        orow[nb] = col.row;
        mask[nb] = col.mask;
        if (wave == nb % W) {                                        // a block's q by one wave
            f4 x[8];
            h8 qh[4], ql[4];
            float unit;
            load_q<CT>(col, g4, x);
            split_q(x, p.scale, unit, qh, ql);
            char * to = lds + nb * 8 * kWave * 16 + lane * 16;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                *reinterpret_cast<h8 *>(to + ks * kWave * 16) = qh[ks];
                *reinterpret_cast<h8 *>(to + (4 + ks) * kWave * 16) = ql[ks];
            }
            if (g4 == 0) *reinterpret_cast<float *>(lds + kWideQ + (nb * 16 + c16) * 4) = unit;
        }
    }
    __syncthreads();
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) c[nb] = *reinterpret_cast<const float *>(lds + kWideQ + (nb * 16 + c16) * 4);
    // steps that every column sees whole
    const int full = TREE ? max(0, min(t.past, t.cap)) / KS : max(0, min(t.past + t.col0 / p.group, t.cap - 1) + 1) / KS;
    [[maybe_unused]] bool small = false;
    float m[NB], l[NB];
    f4 O[NB][8];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        m[nb] = -INFINITY;
        l[nb] = 0.0f;
#pragma unroll
        for (int db = 0; db < 8; ++db) O[nb][db] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // A step; more: the next one's rows are loaded on the way.  Loads under a condition would make every wait one for all loads.
    auto step = [&](auto more) {
        int holes = 0;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            pg[kb] = pg_next[kb];
            holes |= pg[kb] < 0 ? 1 << kb : 0;
        }
        f4 S[NB][KB], key_scale[KB], vs[KB];
        {
            u4 a[8];
            k_step.arrived();
            if constexpr (Q8) {
                u4 rk[4];
#pragma unroll
                for (int f = 0; f < 4; ++f) rk[f] = k_step.chunk(f >> 1, c16, (f & 1) * 4 + g4);
                k_operands(rk, a);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) key_scale[kb] = ks[kb], vs[kb] = vs_next[kb];
            } else {
#pragma unroll
                for (int f = 0; f < 8; ++f) a[f] = k_step.chunk(f >> 2, c16, (f & 3) * 4 + g4);
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                __builtin_amdgcn_sched_barrier(0);                        // q of one block of columns at a time in registers
                const char * from = lds + nb * 8 * kWave * 16 + lane * 16;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) S[nb][kb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int f = 0; f < 8; ++f) {
                    const h8 q = *reinterpret_cast<const h8 *>(from + f * kWave * 16);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
                        S[nb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a[kb * 4 + (f & 3)]), q, S[nb][kb], 0, 0, 0);
                    }
                }
            }
        }
        if constexpr (more.value) {
            place(st + W);
            k_step.read();
            load_k();
        }
        if constexpr (Q8) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) S[nb][kb] *= key_scale[kb];
            }
        }
        if (st >= full || holes != 0) mask_step<NB, KB, TREE>(p, S, lim, mask, t.past, st * KS, g4, holes);
        // rows of keys that no column sees, and of no page, are whatever memory holds: not even 0 times that
        if (st * KS + KS > t.kend || holes != 0) {
#pragma unroll
            for (int f = 0; f < 8; ++f) {
                if (st * KS + v_key<true>(f, g4) >= t.kend || pg[f >> 2] < 0) {
                    if constexpr (Q8) vs[f >> 2][f & 3] = 0.0f;
                    else rv[f] = u4{0, 0, 0, 0};
                }
            }
        }
        float pr[NB][KB][4];
        if constexpr (Q8) {
            weighted_step<NB>(S, vs, c, m, l, O, pr, small);
        } else {
            softmax_step<NB, KB>(S, c, m, l, O, pr);
        }
        h8 ph[NB], pl[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) split_p(pr[nb], ph[nb], pl[nb]);
        u4 vt[2];
#pragma unroll
        for (int db = 0; db < 8; ++db) {
            if constexpr (!Q8) vt[db & 1] = transposed(rv, db);
            else if (db % 4 == 0) v_operands<0>(rv8, db >> 2, vt[0], vt[1]);
            else if (db % 4 == 2) v_operands<1>(rv8, db >> 2, vt[0], vt[1]);
            const h8 a = __builtin_bit_cast(h8, vt[db & 1]);
#pragma unroll
            for (int part = 0; part < 2; ++part) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) O[nb][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, part ? pl[nb] : ph[nb], O[nb][db], 0, 0, 0);
            }
        }
        if constexpr (more.value) {
            load_v();
            entries_of(st + 2 * W, entry);
        }
    };
    for (; st + W < t.step_hi; st += W) step(std::true_type{});
    if (st < t.step_hi) step(std::false_type{});
    float mc[NB];
    uint32_t redo[NB];
    close_columns<NB, false, Q8>(orow, c, m, l, O, mc, redo, small);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        __syncthreads();                                                  // q and the block before are no longer read
        merge_waves<CT, 16, false, TREE, W>(p, t, head, lds, wave, lane, orow[nb], lim[nb], mc[nb], l[nb], O[nb], redo[nb]);
    }
}

// 128 columns of a long chunk on f16 pages: 4 waves of 32 each share the K and V of a tile of keys through LDS, which cuts what
// the CUs pull from L2 to an eighth of what attn_rows' tiles do; for long chunks far behind that traffic sets the pace.  A tile of
// keys is two steps; a step lies in LDS as the MFMA operands themselves, 8 of K and 8 of V^T, 64 lanes x 16 bytes each:
// every read and write is one unbroken kilobyte and no wave rearranges anything.  Waves 0 and 1 fetch and transpose V of
// the two steps, waves 2 and 3 fetch K.  Two tiles in LDS, the next one's rows in registers: one barrier per tile, and two
// workgroups per CU, each multiplying while the other waits at its barrier.  (On f32 pages, whose products take four times
// as long, the same scheme took 101 us against 112 of attn_rows at 300 tokens behind 3500 positions, 281 / 302 at 1024 behind 2889, but
// 88 / 58 at 1024 behind none and 136 / 111 at four of 256 behind 500 to 1500, and attn_rows has become faster since: it takes them all.)
constexpr int kTileSteps = 2;
static_assert(kWaves == 2 * kTileSteps, "a wave fetches K or V of one step");
constexpr int kTileCols = kWaves * 32;
constexpr int kStepBytes = 16 * kWave * 16;   // a step's 16 operands
constexpr size_t kTileLds = 2 * kTileSteps * kStepBytes;
constexpr int kOutStride = kHeadDim + 4, kOutFloats = 16 * kOutStride;   // a wave's 16 columns on their way out
static_assert(kWaves * kOutFloats * sizeof(float) <= kTileLds, "the outputs go through the operands' LDS");

__device__ inline void attn_tile(const AttnParams & p, int block, char * lds) {
    typedef _Float16 CT;
    constexpr bool F16 = true;
    constexpr int KS = step_keys(F16), KB = KS / 16, NB = 2;
    __shared__ int s_holes[2][kTileSteps];                            // bit kb: 16-key block kb of the step lies on no page
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    Tile t;
    int head;
    if (!find_tile<kTileCols, KS, false, false>(p, block, lane, t, head)) return;   // uniform for the workgroup

    // columns: their q is on its way while the first tile is fetched
    int lim[NB], orow[NB];
    f4 x[NB][8];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const Column col = column_of<false>(p, t, head, t.col0 + wave * 16 * NB + nb * 16 + c16);
        lim[nb] = col.lim;
        orow[nb] = col.row;
        load_q<CT>(col, g4, x[nb]);
    }
    // keys that the wave's last and first token see (its columns are in order of token)
    const int first_col = t.col0 + wave * 16 * NB;
    int wave_steps = 0, full = 0;                                     // steps behind the first hold nothing that the wave sees
    if (first_col < t.n_cols) {
        wave_steps = min(t.step_hi, (min(t.past + (min(first_col + 16 * NB, t.n_cols) - 1) / p.group, t.cap - 1) + KS) / KS);
        full = max(0, min(t.past + first_col / p.group, t.cap - 1) + 1) / KS;
    }

    // this wave's share of a tile: K or V of step `mine`
    const bool fetch_v = wave < kTileSteps;
    const int mine = wave & (kTileSteps - 1);
    const HeadRows<CT> rows(p.pages, p.layer, p.n_kv, p.n_pages, p.page_shift, head);
    const int in_page = (1 << p.page_shift) - 1, last_entry = p.seqs.table_stride - 1;
    u4 r[8];
    int pg[KB], entry[KB], st_held = 0;
    auto entries_of = [&](int st) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) entry[kb] = t.table[min((st * KS + kb * 16) >> p.page_shift, last_entry)];
    };
    auto fetch = [&](int st) {
        st_held = st;
        const CT * at[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            pg[kb] = entry_page(p, t, entry[kb], st * KS + kb * 16);
            at[kb] = rows.page(max(pg[kb], 0)) + ((st * KS + kb * 16) & in_page) * kHeadDim + (fetch_v ? rows.v_elems : 0);
        }
#pragma unroll
        for (int f = 0; f < 8; ++f) {
            r[f] = *reinterpret_cast<const u4 *>(at[f >> 2] + (fetch_v ? v_offset<F16>(f, c16, g4) : k_offset(f, c16, g4)));
        }
    };
    auto put = [&](int buf) {
        char * to = lds + (buf * kTileSteps + mine) * kStepBytes + lane * 16;
        if (fetch_v) {
            bool hole = st_held * KS + KS > t.kend;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) hole = hole || pg[kb] < 0;
            if (hole) {   // rows that no column sees, and of no page: not even 0 times what memory holds
#pragma unroll
                for (int f = 0; f < 8; ++f) {
                    if (st_held * KS + v_key<F16>(f, g4) >= t.kend || pg[f >> 2] < 0) r[f] = u4{0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int f = 0; f < 8; ++f) *reinterpret_cast<u4 *>(to + (8 + f) * kWave * 16) = transposed(r, f);
        } else {
#pragma unroll
            for (int f = 0; f < 8; ++f) *reinterpret_cast<u4 *>(to + f * kWave * 16) = r[f];
            if (lane == 0) s_holes[buf][mine] = (pg[0] < 0 ? 1 : 0) | (pg[1] < 0 ? 2 : 0);
        }
    };

    const int n_tiles = (t.step_hi - t.step_lo + kTileSteps - 1) / kTileSteps;
    if (n_tiles > 0) {
        entries_of(t.step_lo + mine);
        fetch(t.step_lo + mine);
        entries_of(t.step_lo + kTileSteps + mine);
    }
    float c[NB];
    h8 qh[NB][4], ql[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        split_q(x[nb], p.scale, c[nb], qh[nb], ql[nb]);
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
    if (n_tiles > 0) {
        put(0);
        fetch(t.step_lo + kTileSteps + mine);
        entries_of(t.step_lo + 2 * kTileSteps + mine);
    }
    __syncthreads();
    for (int tile = 0; tile < n_tiles; ++tile) {
        const char * buf = lds + (tile & 1) * kTileSteps * kStepBytes + lane * 16;
        const int st0 = t.step_lo + tile * kTileSteps;
#pragma unroll 1
        for (int s = 0; s < kTileSteps; ++s) {
            const int st = st0 + s;
            if (st >= wave_steps) break;                              // uniform for the wave
            const char * op = buf + s * kStepBytes;
            u4 a[8], v[8];
#pragma unroll
            for (int f = 0; f < 8; ++f) a[f] = *reinterpret_cast<const u4 *>(op + f * kWave * 16);
            f4 S[NB][KB];
            scores_step<F16, false, NB>(a, qh, ql, x, S);
#pragma unroll
            for (int f = 0; f < 8; ++f) v[f] = *reinterpret_cast<const u4 *>(op + (8 + f) * kWave * 16);
            const int holes = __builtin_amdgcn_readfirstlane(s_holes[tile & 1][s]);
            if (st >= full || holes != 0) mask_step<NB, KB, false>(p, S, lim, lim, t.past, st * KS, g4, holes);
            float pr[NB][KB][4];
            softmax_step<NB, KB>(S, c, m, l, O, pr);
            h8 ph[NB], pl[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) split_p(pr[nb], ph[nb], pl[nb]);
#pragma unroll
            for (int part = 0; part < 2; ++part) {
#pragma unroll
                for (int db = 0; db < 8; ++db) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        O[nb][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, v[db]), part ? pl[nb] : ph[nb], O[nb][db], 0, 0, 0);
                    }
                }
            }
        }
        if (tile + 1 < n_tiles) {
            put((tile + 1) & 1);
            if (tile + 2 < n_tiles) {
                fetch(st0 + 2 * kTileSteps + mine);
                entries_of(st0 + 3 * kTileSteps + mine);
            }
        }
        __syncthreads();
    }
    float mc[NB];
    uint32_t redo[NB];
    close_columns<NB, false, false>(orow, c, m, l, O, mc, redo, false);
    // through the wave's own part of LDS, so that a store instruction writes two whole rows; a lane's values would lie 16 bytes
    // in each of 64 lines
    float * so = reinterpret_cast<float *>(lds) + wave * kOutFloats;
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
            if (row >= 0 && !((redo[nb] >> col) & 1)) store_column<false>(p, t, row, lm, dim, v, cm, cl, dim == 0);
        }
        redo_columns<CT, KS>(p, t, head, lane, lim[nb], orow[nb], redo[nb]);
    }
}

// The launches.  One kind of tile, or longer chunks first and the sequences of few columns behind them.
// Registers are cut for three waves per SIMD, or one workgroup of 8 waves per CU.
template <typename CT, bool FEW, bool TREE, int W>
__global__ __launch_bounds__(W * kWave, W > kWaves ? 2 : 3) void paged_rows_kernel(AttnParams p) {
    extern __shared__ __attribute__((aligned(16))) char lds_rows[];
    attn_rows<CT, FEW, TREE, W>(p, blockIdx.x, lds_rows);
}

template <typename CT, bool TREE>
__global__ __launch_bounds__(kThreads, 3) void paged_rows_both_kernel(AttnParams p) {
    extern __shared__ __attribute__((aligned(16))) char lds_rows[];
    const int many = p.tiles_many * p.n_kv * p.splits_many, block = blockIdx.x;
    if (block < many) attn_rows<CT, false, TREE, kWaves>(p, block, lds_rows);
    else attn_rows<CT, true, TREE, kWaves>(p, block - many, lds_rows);
}

template <typename CT, bool TREE, int W>
__global__ __launch_bounds__(W * kWave, 2) void paged_wide_kernel(AttnParams p) {
    extern __shared__ __attribute__((aligned(16))) char lds_wide[];
    attn_wide<CT, TREE, W>(p, blockIdx.x, lds_wide);
}

template <bool BOTH>
__global__ __launch_bounds__(kThreads, 2) void paged_tile_kernel(AttnParams p) {
    extern __shared__ __attribute__((aligned(16))) char lds_tile[];
    const int many = p.tiles_many * p.n_kv * p.splits_many, block = blockIdx.x;
    if (!BOTH || block < many) attn_tile(p, block, lds_tile);
    else attn_rows<_Float16, true, false, kWaves>(p, block - many, lds_tile);
}

// Joins the splits of each (row, head): one wave each, lane = split for the weights, then lane = 2 dims.  Its time is
// dependent loads, so the sequences, the weights and the first results are read together; a split that the row does not
// reach holds whatever the workspace held, and is selected away.
template <bool TREE, int kFirst>
__global__ __launch_bounds__(256) void paged_join_kernel(AttnParams p, int ks) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= static_cast<int64_t>(p.seqs.n_rows) * p.n_heads) return;
    const int row = static_cast<int>(item / p.n_heads);
    const float * po = p.part_o + item * p.n_parts * kHeadDim + 2 * lane;
    f2 ml = p.part_ml[item * p.n_parts + min(lane, p.n_parts - 1)];
    f2 part[kFirst];
#pragma unroll
    for (int s = 0; s < kFirst; ++s) part[s] = *reinterpret_cast<const f2 *>(po + min(s, p.n_parts - 1) * kHeadDim);
    const RowPlace at = row_place(p.seqs, row, lane);
    if (at.seq < 0) return;
    const bool few = at.rows * p.group <= p.few_max;
    const int n_splits = few ? p.splits_few : p.splits_many, split_steps = few ? p.steps_few : p.steps_many;
    if (n_splits == 1) return;                                        // stored by its tile
    const int cap = p.seqs.table_stride << p.page_shift;
    const int lim = min(TREE ? at.past + at.rows - 1 : at.pos, cap - 1);
    // splits that hold a key which this row sees (the first is always computed)
    const int active = lim < 0 ? 1 : min(n_splits, lim / ks / split_steps + 1);
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
    const float inv = inverse_sum<TREE>(p, p.seqs.tables + static_cast<int64_t>(at.seq) * p.seqs.table_stride, lim, at.past, static_cast<int>(item), L);
    *reinterpret_cast<f2 *>(p.out + item * kHeadDim + 2 * lane) = o * inv;
}

// How a call cuts its work: which kinds of tiles there are, their upper bounds, and the key ranges of each kind.
struct AttnPlan {
    bool tile;               // the longer sequences' tiles are attn_tile's
    bool wide;               // or attn_wide's
    bool eight;              // of 8 waves per workgroup
    int tiles_many, tiles_few;
    int few_max;             // 0: sequences of few columns are the longer ones' tiles, too
    int splits_many, splits_few, steps_many, steps_few;
    int parts() const { return std::max(splits_many, splits_few); }
};

// Key ranges of `steps` steps for workgroups of which one range has `blocks`: enough to make `target` of them, of `least` steps or
// so, and more than one only where there are twice as many: two of 5 or 7 steps lose more to the join than they gain (one
// token behind 400 positions 9.7 us, in one range 8.4, both before K went through LDS; 128 tokens behind 500, `least` 16, 12.7 and 8.9).
void cut_keys(int steps, int64_t blocks, int64_t target, int64_t least, int64_t most, int & splits, int & split_steps) {
    const int64_t by_length = steps < 2 * least ? 1 : (steps + least - 1) / least;
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>({target / std::max<int64_t>(blocks, 1), by_length, most}));
    split_steps = std::max<int>(1, static_cast<int>((steps + n - 1) / n));
    splits = std::max(1, (steps + split_steps - 1) / split_steps);
}

AttnPlan attn_plan(const qa_kv_layout & l, const qa_paged_batch & b, int32_t n_heads, size_t workspace_bytes, bool tree) {
    const bool f16 = l.cache_type != QA_CACHE_F32;                    // products
    const int ks = step_keys(f16);
    const int group = n_heads / l.n_kv_heads;
    const int seqs = std::min(b.n_seqs, b.n_rows);
    const int64_t tokens = std::min<int64_t>(b.n_rows, b.max_tokens > 0 ? b.max_tokens : b.n_rows);
    const int64_t most = tokens * group, cols = static_cast<int64_t>(b.n_rows) * group;   // columns of a sequence, of all
    const int64_t cap = static_cast<int64_t>(b.table_stride) * l.max_seq;
    const int64_t len = std::min<int64_t>(cap, b.max_len > 0 ? b.max_len : cap);
    const int steps = static_cast<int>((len + ks - 1) / ks);
    const size_t per_part = static_cast<size_t>(b.n_rows) * n_heads * (kHeadDim + 2) * sizeof(float);
    const int64_t parts = std::min<int64_t>(kMaxSplits, std::max<size_t>(1, workspace_bytes / per_part));
    AttnPlan pl{};
    const bool many = most > few_cols(f16);
    // attn_tile (causal, f16 pages) against attn_rows: by the products, where a sequence fills three tiles, so that a batch keeps the
    // kernel, and the bits, that it had before attn_rows took K through LDS.  Since then, us: 1024 tokens behind 2889 positions
    // 76 / 78, behind 8000 146 / 180, three of 1024 behind 2889 247 / 264, but 256 behind 3000 37 / 27, 700 behind 1500 45 / 35; 512
    // behind 1000 33 / 20, 1024 behind none 37 / 24, eight of 100 behind 2000 (columns left empty) 59 / 39, which it leaves to attn_rows.
    const bool fresh = tree || l.cache_type == QA_CACHE_Q8;
    pl.tile = f16 && !fresh && most > 2 * kTileCols && cols * (len - std::min(len, tokens / 2)) > 1600000;
    // one sequence is of one kind; of several at most few_seqs are of few columns, by the host's counts
    const int64_t few_tokens = few_cols(f16) / group;
    const int64_t few_seqs = tokens > few_tokens ? (seqs * tokens - b.n_rows) / (tokens - few_tokens) : seqs;
    const bool few = !many || (b.n_seqs > 1 && (!fresh || 4 * few_seqs >= 3 * seqs));
    int64_t eight_tiles = 0;
    if (fresh && !few && most > 16) {
        // 8 bits and trees on 8 KV heads, us.  One workgroup of 8 waves per CU, where the tiles and their ranges fill 166 of the 256 CUs, or 120 of
        // them for 40 steps at most, and each has enough to do for what it takes to begin and to merge (`worth`): sixteen trees of up to 41
        // behind 156 to 3000 in attn_wide of 8 / 4 waves and in attn_rows 37 / 44 / 45, five behind 1600 18.5 / 20.9 / 20.6, but one
        // of 64 behind 3000 15.9 / 16.6 / 15.1, six of up to 20 behind 500 to 1500 16.3 / 16.8 / 15.3; two of 63 in f32 with attn_rows
        // of 8 / 4 waves 20 / 24.  8 bits: 64 tokens behind 3000 16.3 / 17.3 / 17.0, two trees of 32 behind 2000 16.5 / 17.5 / 16.5, sixteen of
        // 1 to 12 behind 300 to 2000 (tiles mostly empty) 20.9 / 21.7 / 19.5, 300 tokens (152 tiles) behind 3500 38.5 / 35.6 / 48.
        // More tiles, or few: attn_wide for long products (1024 tokens behind 2889 73, attn_rows 85, behind none 21 / 24, 24 trees of 64
        // behind 1000 to 3000 69 / 78), attn_rows for short ones (32 trees of up to 41 behind 156 to 1000 on 8 bits 27 / 25).
        // a sequence's last tile is half full
        const int64_t columns = f16 ? kWideCols : 16, t = std::max<int64_t>((cols + columns - 1) / columns + (seqs - 1) / 2, seqs) * l.n_kv_heads;
        const int64_t ranges = std::min<int64_t>(256 / std::min<int64_t>(t, 256), (steps + 15) / 16);
        const bool fills = t <= 256 && t * ranges >= (steps <= 40 * ranges ? 120 : 166);
        const bool worth = !f16 || (l.cache_type == QA_CACHE_Q8 ? cols * len >= 300000 && cols >= 24 * seqs : cols * len >= 400000);
        pl.eight = fills && worth;
        eight_tiles = t;
        pl.wide = f16 && (pl.eight || cols * len >= 2000000);
    }
    const int width = pl.tile ? kTileCols : pl.wide ? kWideCols : 16;
    pl.tiles_many = many ? static_cast<int>(cols / width + seqs) : 0;
    pl.few_max = few ? few_cols(f16) : 0;
    pl.tiles_few = few ? seqs : 0;
    // Workgroups to make of the keys, us.  Decode steps, and sequences of one tile: K and V are what they read, and more, shorter
    // ranges keep more of them in flight.  Longer ones read K and V once per tile, from L2, and every range writes and reads its
    // columns' partial results: 256 tokens behind 1000 positions (256 tiles) in 1 / 2 / 3 ranges 12.1 / 17.4 / 20.0 (f32 pages 28.7 / 32.6 /
    // 35.4), 64 behind 3000 (64 tiles) in 4 / 6 / 8 17.5 / 16.2 / 18.2 (34.7 / 27.8 / 30.5).  With few CUs left over by the tiles of a long
    // context their partial results cost less than the wait for the CUs that have one more: 300 behind 3500 (304 tiles) on f32
    // pages 124 in one, 98 in two, 92 in three.  Sequences differ in length, and the ranges are cut for the longest: 16 of 70 behind 300
    // to 2000, 1 / 2 / 3 ranges 64 / 67 / 70 (f32, which takes one, too, 140 / 132 / 134).  attn_tile has 512 workgroups at a time: 400
    // behind 3500 in 3 / 4 / 9 ranges 64 / 54 / 46, two of 600 and eight of one token behind 24 to 3500 in 3 / 4 / 5 / 6 93 / 78 / 77 / 78, but
    // four of 256 behind 500 to 1500, which get six, in 3 / 4 / 6 60 / 53 / 59.  128 behind 500 on f32 pages get three, 18.6, one is 16.8.
    const int64_t heads = static_cast<int64_t>(seqs) * l.n_kv_heads;
    const int64_t tiles = pl.eight ? eight_tiles : std::max<int64_t>(1, (cols + width - 1) / width) * l.n_kv_heads;
    const bool one = b.n_seqs == 1;
    // one round of workgroups where their ranges stay short: four sequences of 501 to 3001 in 8 / 12 ranges 13.3 / 16.2 us, f32 pages 18.3 / 23.6
    const int64_t round = std::max<int64_t>(1, 256 / heads), decode = (steps + round - 1) / round <= 24 ? 256 : 1024;
    if (fresh && most > 16) cut_keys(steps, tiles, pl.eight ? 256 : one && !pl.wide ? 384 : few ? 640 : 512, 16, parts, pl.splits_many, pl.steps_many);
    else if (pl.tile) cut_keys(steps, tiles, one ? 512 : 768, 4, parts, pl.splits_many, pl.steps_many);
    else if (most <= 16) cut_keys(steps, heads, decode, 8, parts, pl.splits_many, pl.steps_many);
    else cut_keys(steps, tiles, !one ? 640 : steps >= 128 && tiles > 192 ? 1024 : 384, 16, parts, pl.splits_many, pl.steps_many);
    cut_keys(steps, heads, decode, 8, parts, pl.splits_few, pl.steps_few);
    if (!many) pl.splits_many = 1;
    if (!few) pl.splits_few = 1;
    return pl;
}

template <bool TREE>
void launch_join(const AttnParams & p, bool f16, hipStream_t stream) {
    const int64_t items = static_cast<int64_t>(p.seqs.n_rows) * p.n_heads;
    const auto kernel = p.n_parts <= 2 ? &paged_join_kernel<TREE, 2> : &paged_join_kernel<TREE, 8>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256), 0, stream, p, step_keys(f16));
}

// Decode steps on f16 pages run with three workgroups per CU and the others behind them, where registers would allow four: sequences of
// uneven lengths gain more than those of one length lose.  Behind 156 to 3900 positions, three / four: eight 19.9 / 21.7 us, sixteen
// 28.1 / 31.3, 32 48.5 / 54.8, 64 94.4 / 93.3; 32 behind 1000 to 3000 49.7 / 50.1; of the same length 32 behind 1000 27.8 / 26.6, 64 46.0 / 45.8,
// 16 and 32 behind 3900 the same.  (Two per CU: 52.6 for the 32.)  LDS keeps the fourth out.  The other few-column kernels' registers
// are for three as it is.
constexpr size_t kThreePerCu = 41 * 1024;

// The longer sequences' kernel, or both kinds' in one launch.
template <typename CT, bool TREE>
int launch_attn(const AttnPlan & pl, AttnParams p, hipStream_t stream) {
    constexpr bool F16 = f16_products<CT>, FRESH = TREE || is_q8<CT>;
    const dim3 grid(static_cast<unsigned>(p.n_kv) * (pl.tiles_many * pl.splits_many + pl.tiles_few * pl.splits_few));
    constexpr size_t lds_few = rows_bytes<CT>(true), lds_many = rows_bytes<CT>(false);
    static_assert(lds_few <= kTileLds && lds_few <= lds_many, "a launch of both kinds has the longer ones' LDS");
    auto kernel = !pl.tiles_many ? &paged_rows_kernel<CT, true, TREE, kWaves>
                  : pl.few_max ? &paged_rows_both_kernel<CT, TREE> : &paged_rows_kernel<CT, false, TREE, kWaves>;
    size_t lds = pl.tiles_many ? lds_many : F16 && !FRESH ? std::max(lds_few, kThreePerCu) : lds_few;
    int waves = kWaves;
    if constexpr (F16 && FRESH) {
        if (pl.wide) {
            kernel = pl.eight ? &paged_wide_kernel<CT, TREE, 8> : &paged_wide_kernel<CT, TREE, kWaves>;
            waves = pl.eight ? 8 : kWaves;
            lds = wide_lds<CT>(waves);
        }
    } else if constexpr (FRESH) {
        if (pl.eight) {
            kernel = &paged_rows_kernel<CT, false, TREE, 8>;
            waves = 8;
            lds = rows_bytes<CT>(false, waves);
        }
    } else if constexpr (F16) {
        if (pl.tile) {
            kernel = pl.few_max ? &paged_tile_kernel<true> : &paged_tile_kernel<false>;
            lds = kTileLds;
        }
    }
    if (lds >= kTileLds) {
        QA_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
    }
    hipLaunchKernelGGL(kernel, grid, dim3(static_cast<unsigned>(waves * kWave)), lds, stream, p);
    QA_LAUNCH_CHECK("paged attention kernel");
    if (pl.parts() > 1) {
        launch_join<TREE>(p, F16, stream);
        QA_LAUNCH_CHECK("paged_join_kernel");
    }
    return QA_OK;
}

template <bool TREE>
int launch_typed(const AttnPlan & pl, const AttnParams & p, int32_t cache_type, hipStream_t stream) {
    if (cache_type == QA_CACHE_Q8) return launch_attn<int8_t, TREE>(pl, p, stream);
    if (cache_type == QA_CACHE_F16) return launch_attn<_Float16, TREE>(pl, p, stream);
    return launch_attn<float, TREE>(pl, p, stream);
}

// mask null: causal.
int attention(const float * q, const void * pages, const qa_kv_layout * layout, int32_t layer, const qa_paged_batch * batch,
              const uint32_t * mask, int32_t mask_words, int32_t n_heads, float scale, float * out, void * workspace,
              size_t workspace_bytes, void * stream, const char * name) {
    const std::string who = name;
    if (check_batch(layout, layer, batch, n_heads, name) != QA_OK) return QA_ERR_INVALID;
    if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(QA_ERR_INVALID, who + ": scale must be positive and finite");
    if (batch->n_rows == 0) return QA_OK;
    if (!q || !pages || !out || (!workspace && workspace_bytes > 0)) return fail(QA_ERR_INVALID, who + ": null pointer");
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(out) |
          reinterpret_cast<uintptr_t>(workspace)) & 15) != 0) {
        return fail(QA_ERR_INVALID, who + ": pointers must be aligned to 16 bytes");
    }
    if (static_cast<int64_t>(batch->n_rows) * n_heads > INT32_MAX / 2) return fail(QA_ERR_INVALID, who + ": too many rows");
    if (const int rc = check_stream(stream, name); rc != QA_OK) return rc;
    const AttnPlan pl = attn_plan(*layout, *batch, n_heads, workspace_bytes, mask != nullptr);
    if ((static_cast<int64_t>(pl.tiles_many) * pl.splits_many + static_cast<int64_t>(pl.tiles_few) * pl.splits_few) * layout->n_kv_heads > INT32_MAX / kThreads) {
        return fail(QA_ERR_INVALID, who + ": too many rows");
    }
    AttnParams p{};
    p.q = q;
    p.pages = pages;
    p.out = out;
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = reinterpret_cast<f2 *>(p.part_o + static_cast<int64_t>(batch->n_rows) * n_heads * pl.parts() * kHeadDim);
    p.seqs = paged_seqs(*batch);
    p.n_heads = n_heads;
    p.n_kv = layout->n_kv_heads;
    p.group = n_heads / layout->n_kv_heads;
    p.n_pages = layout->n_streams;
    p.page_shift = page_shift_of(layout->max_seq);
    p.layer = layer;
    p.few_max = pl.few_max;
    p.tiles_many = pl.tiles_many;
    p.tiles_few = pl.tiles_few;
    p.splits_many = pl.splits_many;
    p.splits_few = pl.splits_few;
    p.steps_many = pl.steps_many;
    p.steps_few = pl.steps_few;
    p.n_parts = pl.parts();
    p.scale = scale;
    p.mask = mask;
    p.mask_words = mask_words;
    return mask ? launch_typed<true>(pl, p, layout->cache_type, as_stream(stream))
                : launch_typed<false>(pl, p, layout->cache_type, as_stream(stream));
}

}  // namespace
}  // namespace qa

extern "C" size_t qa_paged_attn_workspace_bytes(const qa_kv_layout * layout, const qa_paged_batch * batch, int32_t n_heads) {
    using namespace qa;
    if (check_batch_sizes(layout, 0, batch, n_heads, "qa_paged_attn_workspace_bytes") != QA_OK || batch->n_rows == 0) return 0;
    // causal or a tree: enough for either
    const int parts = std::max(attn_plan(*layout, *batch, n_heads, SIZE_MAX, false).parts(), attn_plan(*layout, *batch, n_heads, SIZE_MAX, true).parts());
    if (parts <= 1) return 0;
    return static_cast<size_t>(batch->n_rows) * n_heads * parts * (kHeadDim + 2) * sizeof(float);
}

extern "C" int qa_paged_attn(const float * q, const void * pages, const qa_kv_layout * layout, int32_t layer,
                             const qa_paged_batch * batch, int32_t n_heads, float scale, float * out, void * workspace,
                             size_t workspace_bytes, void * stream) {
    return qa::attention(q, pages, layout, layer, batch, nullptr, 0, n_heads, scale, out, workspace, workspace_bytes, stream, "qa_paged_attn");
}

extern "C" int qa_paged_tree_attn(const float * q, const void * pages, const qa_kv_layout * layout, int32_t layer,
                                  const qa_paged_batch * batch, const uint32_t * mask, int32_t mask_words, int32_t n_heads, float scale,
                                  float * out, void * workspace, size_t workspace_bytes, void * stream) {
    using namespace qa;
    const char * who = "qa_paged_tree_attn";
    if (check_batch(layout, layer, batch, n_heads, who) != QA_OK || check_tree(batch, mask_words, who) != QA_OK) return QA_ERR_INVALID;
    if (batch->n_rows > 0 && !mask) return fail(QA_ERR_INVALID, "qa_paged_tree_attn: null pointer");
    return attention(q, pages, layout, layer, batch, mask, mask_words, n_heads, scale, out, workspace, workspace_bytes, stream, who);
}
