// Beam search: the best continuations over a group's beams and the vocabulary, and the beams' states put in their new order.
//
// Selection in two launches.  The first streams the logits once (a wave takes a unit of a row, values in registers): the largest
// value of every 256, and the unit's maximum and sum of exponentials.  The second, a workgroup per group, needs no more than
// those: a row's logarithm of its sum turns maxima into scores, and the new beams are among the values of the `width` best
// 256s, as any value outside has `width` better ones (of 256s that tie, the earlier has the lower ids).  It reads those again,
// width x 1 KB.  Both of its choices, of 256s and of values, go the same way: a bound that at least `width` entries
// reach, a list of the entries that reach it, and each entry's rank in the list by counting.
// Exponentials are f32, sums and scores f64, so that candidates of different beams compare as in the formula.
#include "common.hpp"
#include "paged.hpp"
#include "wave.hpp"

#include <algorithm>

namespace qa {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // rows of an odd vocabulary start anywhere

constexpr int kSeg = 256;            // values per maximum: a wave's load
constexpr int kMaxWidth = 64;
constexpr int kMaxStops = 64;
constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / kWave;
constexpr int kListMax = 1024;       // entries that reach the bound; more are taken one by one

struct Unit {
    double sum;      // of exp(x - most)
    float most, pad;
};

struct BeamParams {
    const float * logits;
    const float * scores;
    const int32_t * done;
    const int32_t * stop_ids;
    int32_t * parents;
    int32_t * tokens;
    float * scores_out;
    int32_t * done_out;
    Unit * units;        // [rows][n_units]
    float * seg_max;     // [rows][n_segs]
    int32_t width, vocab, n_stop, n_units, n_segs;
};

// 2^t to 2^-23 of itself: what t loses as an f32 goes in behind the instruction.  (A difference x - most rounded to f32 would be off by
// 2^-24 |x - most|, the same way for many equal values.)
constexpr double kLog2e = 1.4426950408889634;
__device__ inline float exp2_of(double t) {
    const float hi = static_cast<float>(t), lo = static_cast<float>(t - static_cast<double>(hi));
    const float e = __builtin_amdgcn_exp2f(hi);
    return hi > -INFINITY ? fmaf(e * lo, 0.6931472f, e) : 0.0f;
}

// 512 values per wave: 64 rows of 151936 in 1, 2, 4 and 8 loads per lane 13, 9.7, 10.8 and 12.3 us (read at 4 TB/s; a wave's
// instructions take as long as its values, and short waves overlap the two), 4 rows 3.0 in 2 and 4.5 in 8.
constexpr int kLoads = 2;
__global__ __launch_bounds__(256) void beam_units_kernel(BeamParams p) {
    const int lane = threadIdx.x & (kWave - 1);
    const int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.y;
    if (unit >= p.n_units || (p.done && p.done[row] != 0)) return;       // a beam that is done has one candidate
    const float * x = p.logits + static_cast<int64_t>(row) * p.vocab;
    const int first = unit * kLoads * 256 + lane * 4;
    f4u v[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
        const int at = first + u * 256;
        if (at + 4 <= p.vocab) {
            v[u] = *reinterpret_cast<const f4u *>(x + at);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] = at + e < p.vocab ? x[at + e] : -INFINITY;
        }
    }
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
        float seg = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[u][e] = fmaxf(v[u][e], -INFINITY);           // NaN: none
            seg = fmaxf(seg, v[u][e]);
        }
        seg = wave_max_all(seg);
        const int s = unit * kLoads + u;
        if (lane == 0 && s < p.n_segs) p.seg_max[static_cast<int64_t>(row) * p.n_segs + s] = seg;
        most = fmaxf(most, seg);
    }
    double sum = 0.0;
    if (most > -INFINITY) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += static_cast<double>(exp2_of((static_cast<double>(v[u][e]) - most) * kLog2e));
        }
    }
    sum = wave_sum_d_all(sum);
    if (lane == 0) p.units[static_cast<int64_t>(row) * p.n_units + unit] = Unit{sum, most, 0.0f};
}

// A candidate: its score, and its beam and place, which settle ties: the lower first.
struct Entry {
    double score;
    uint64_t at;
};
__device__ inline uint64_t place_of(int beam, int place) { return (static_cast<uint64_t>(beam) << 32) | static_cast<uint32_t>(place); }
__device__ inline bool better(const Entry & a, const Entry & b) { return a.score > b.score || (a.score == b.score && a.at < b.at); }

// log x of a sum, to 2^-24: the mantissa's in f32.  (In f64 throughout the workgroup waited 1 us for it.)
__device__ inline double log_of(double x) {
    int e;
    const double m = frexp(x, &e);
    return e * 0.6931471805599453 + static_cast<double>(logf(static_cast<float>(m)));
}

struct PickLds {
    double off[kMaxWidth];           // what a row's values are raised by to become scores; -inf: none of them counts
    double stay[kMaxWidth];          // the score of a beam that is done
    Entry list[kListMax];
    Entry chosen[kMaxWidth];
    Entry wave[kPickWaves];
    double sum[kMaxWidth];           // of a beam's exponentials, less its largest value
    float most[kMaxWidth];
    float row_most[4 * kMaxWidth];   // the largest maximum of every 16 lanes, a wave's (or a beam's) four together
    double bound;
    int count;
};

// The `width` best of the list, best first, into chosen: an entry's place is the number of better ones, which 8 lanes count.
__device__ inline void rank_list(PickLds & s, int count, int width) {
    constexpr int kLanes = 8;
    for (int first = 0; first < count; first += kPickThreads / kLanes) {
        const int i = first + static_cast<int>(threadIdx.x) / kLanes;
        const Entry e = s.list[min(i, count - 1)];
        int rank = 0;
        for (int k = threadIdx.x & (kLanes - 1); k < count; k += kLanes) rank += better(s.list[k], e);
        rank += __builtin_amdgcn_mov_dpp(rank, 0xB1, 0xf, 0xf, false);
        rank += __builtin_amdgcn_mov_dpp(rank, 0x4E, 0xf, 0xf, false);
        rank += __builtin_amdgcn_mov_dpp(rank, 0x141, 0xf, 0xf, false);
        if (i < count && rank < width && (threadIdx.x & (kLanes - 1)) == 0) s.chosen[rank] = e;
    }
    __syncthreads();
}

// The same where more entries reach the bound than the list holds (many ties): one after another, each the best of those behind
// the one before.  entry(i) is the i-th of n.
template <typename F>
__device__ inline void one_by_one(PickLds & s, int width, int n, F && entry) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    Entry last{INFINITY, 0};
    for (int r = 0; r < width; ++r) {
        Entry best{-INFINITY, ~uint64_t{0}};
        for (int i = threadIdx.x; i < n; i += kPickThreads) {
            const Entry e = entry(i);
            if (e.score > -INFINITY && better(last, e) && better(e, best)) best = e;
        }
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const Entry o{__shfl_xor(best.score, d, kWave), static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(best.at), d, kWave))};
            if (better(o, best)) best = o;
        }
        if (lane == 0) s.wave[wave] = best;
        __syncthreads();
        last = s.wave[0];
        for (int w = 1; w < kPickWaves; ++w) {
            if (better(s.wave[w], last)) last = s.wave[w];
        }
        if (threadIdx.x == 0) s.chosen[r] = last;
        __syncthreads();
    }
}

// Its time is one workgroup's latencies, and fetching its instructions: short loops, and little that is unrolled.  A wave takes the
// 256s of one beam (or a part of them, for up to 8 beams; or of several beams, one after another, for more than 16), so that it
// looks at maxima as they are, one comparison each, and only what may count becomes a score in 64 bits.  Up to kKeep maxima per
// lane are fetched before the row's sums are added and stay in registers for the second look.  A vocabulary of 151936 takes 7.6 us for
// four beams and 9.0 for eight groups of eight; one maximum per 512 (half as many, and twice the values to read again) 0.4 less for
// eight beams and 1.0 more for 32.
constexpr int kKeep = 10;
static_assert(kPickThreads == 4 * 4 * kMaxWidth, "four lanes rank each of the rows' maxima");

__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(BeamParams p) {
    __shared__ PickLds s;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row0 = blockIdx.x * p.width;
    const int parts = max(1, kPickWaves / p.width), stride = parts * kWave, per_lane = (p.n_segs + stride - 1) / stride;
    const int tasks = p.width * parts;
    const bool keep = tasks <= kPickWaves && per_lane <= kKeep;
    // kKeep maxima of a task, from its lanes' first one behind `from` on
    float held[kKeep];
    auto fetch = [&](int task, int from) {
        const float * maxima = p.seg_max + static_cast<int64_t>(row0 + task / parts) * p.n_segs;
#pragma unroll
        for (int k = 0; k < kKeep; ++k) {
            const int seg = task % parts * kWave + lane + (from + k) * stride;
            held[k] = seg < p.n_segs ? maxima[seg] : -INFINITY;
        }
    };
    if (keep && wave < tasks) fetch(wave, 0);
    // a lane per beam
    double score = -INFINITY;
    bool done = false;
    if (wave == 0 && lane < p.width) {
        score = static_cast<double>(p.scores[row0 + lane]);
        done = p.done && p.done[row0 + lane] != 0;
    }
    if (threadIdx.x == 0) s.count = 0;
    for (int task = wave; task < tasks; task += kPickWaves) {
        const int b = task / parts;
        float most = -INFINITY;
        for (int from = 0; from < per_lane; from += kKeep) {
            if (!keep) fetch(task, from);
#pragma unroll
            for (int k = 0; k < kKeep; ++k) most = fmaxf(most, held[k]);
        }
        most = fmaxf(most, dpp_f<0xB1>(most));
        most = fmaxf(most, dpp_f<0x4E>(most));
        most = fmaxf(most, dpp_f<0x141>(most));
        most = fmaxf(most, dpp_f<0x140>(most));
        if ((lane & 15) == 0) s.row_most[task * 4 + (lane >> 4)] = most;
        if (task % parts != 0) continue;
        // the row's sum
        const Unit * units = p.units + static_cast<int64_t>(row0 + b) * p.n_units;
        constexpr int kUnits = 5;                          // per lane in registers: 320 of a row
        Unit u[kUnits];
        float all = -INFINITY;
#pragma unroll
        for (int k = 0; k < kUnits; ++k) u[k] = units[min(lane + k * kWave, p.n_units - 1)];
#pragma unroll
        for (int k = 0; k < kUnits; ++k) all = fmaxf(all, u[k].most);
        for (int i = lane + kUnits * kWave; i < p.n_units; i += kWave) all = fmaxf(all, units[i].most);
        all = wave_max_all(all);
        double sum = 0.0;
        auto add = [&](const Unit & x) {
            if (x.most > -INFINITY) sum += x.sum * static_cast<double>(exp2_of((static_cast<double>(x.most) - all) * kLog2e));
        };
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            if (lane + k * kWave < p.n_units) add(u[k]);
        }
        for (int i = lane + kUnits * kWave; i < p.n_units; i += kWave) add(units[i]);
        sum = wave_sum_d_all(sum);
        if (lane == 0) {
            s.sum[b] = sum;
            s.most[b] = all;
        }
    }
    // what a beam's values are raised by: one wave for all beams
    __syncthreads();
    if (wave == 0 && lane < p.width) {
        const bool counts = score > -INFINITY && score < INFINITY;
        const float most = s.most[lane];
        s.stay[lane] = counts && done ? score : -INFINITY;
        s.off[lane] = counts && !done && most > -INFINITY && most < INFINITY ? score - (log_of(s.sum[lane]) + most) : -INFINITY;
    }
    __syncthreads();
    // The bound: of those best of 16 lanes each (a beam that is done is one of them), the width-th.
    auto row_best = [&](int i) {
        const int b = (i >> 2) / parts;
        const double off = s.off[b];
        return off > -INFINITY ? off + static_cast<double>(s.row_most[i]) : i == b * parts * 4 ? s.stay[b] : -INFINITY;
    };
    if (static_cast<int>(threadIdx.x) < tasks * 4) s.list[threadIdx.x].score = row_best(threadIdx.x);
    __syncthreads();
    {
        const int i = threadIdx.x >> 2;
        const double v = s.list[min(i, tasks * 4 - 1)].score;
        int rank = 0;
#pragma unroll 4
        for (int j = threadIdx.x & 3; j < tasks * 4; j += 4) {
            const double o = s.list[j].score;
            rank += o > v || (o == v && j < i);
        }
        rank += __builtin_amdgcn_mov_dpp(rank, 0xB1, 0xf, 0xf, false);
        rank += __builtin_amdgcn_mov_dpp(rank, 0x4E, 0xf, 0xf, false);
        if (i < tasks * 4 && rank == p.width - 1 && (threadIdx.x & 3) == 0) s.bound = v;
    }
    __syncthreads();
    double bound = s.bound;
    auto list = [&](const Entry & e) {
        if (!(e.score > -INFINITY) || e.score < bound) return;
        const int to = atomicAdd(&s.count, 1);
        if (to < kListMax) s.list[to] = e;
    };
    for (int task = wave; task < tasks; task += kPickWaves) {
        const int b = task / parts;
        const double off = s.off[b];
        if (!(off > -INFINITY)) continue;
        // What a maximum needs, less what is rounded on the way: a score and the difference to 2^-53 of what they come from, which may
        // be far larger than the difference, and the f32 to 2^-24 of itself.  list() compares the scores.
        const double near = bound - off;
        const float least = static_cast<float>(near - (fabs(near) * 0x1p-22 + (fabs(bound) + fabs(off)) * 0x1p-51));
        for (int from = 0; from < per_lane; from += kKeep) {
            if (!keep) fetch(task, from);
            unsigned some = 0;
#pragma unroll
            for (int k = 0; k < kKeep; ++k) some |= held[k] >= least ? 1u << k : 0u;
            for (; some != 0; some &= some - 1) {          // few
                const int at = __ffs(some) - 1;
                float v = held[0];
#pragma unroll
                for (int k = 1; k < kKeep; ++k) v = k == at ? held[k] : v;
                list(Entry{off + static_cast<double>(v), place_of(b, task % parts * kWave + lane + (from + at) * stride + 1)});
            }
        }
    }
    if (static_cast<int>(threadIdx.x) < p.width) list(Entry{s.stay[threadIdx.x], place_of(threadIdx.x, 0)});
    __syncthreads();
    int count = s.count;
    if (count <= kListMax) {
        rank_list(s, count, p.width);
    } else {
        const int n = p.width * p.n_segs;
        one_by_one(s, p.width, n + p.width, [&](int i) {
            if (i >= n) return Entry{s.stay[i - n], place_of(i - n, 0)};
            const int b = i / p.n_segs, seg = i - b * p.n_segs;
            const double off = s.off[b];
            return Entry{off > -INFINITY ? off + static_cast<double>(p.seg_max[static_cast<int64_t>(row0) * p.n_segs + i]) : -INFINITY, place_of(b, seg + 1)};
        });
    }
    const int n_segs = min(count, p.width);
    // The values of the chosen 256s: those that reach the last one's maximum are at least as many, if there are `width` 256s.
    bound = n_segs == p.width ? s.chosen[n_segs - 1].score : -INFINITY;
    auto value = [&](const Entry * segs, int i) {
        const Entry seg = segs[i / kSeg];
        const int b = static_cast<int>(seg.at >> 32), place = static_cast<int>(static_cast<uint32_t>(seg.at));
        if (place == 0) return Entry{i % kSeg == 0 ? seg.score : -INFINITY, seg.at};
        const int id = (place - 1) * kSeg + i % kSeg;
        const float x = id < p.vocab ? p.logits[static_cast<int64_t>(row0 + b) * p.vocab + id] : -INFINITY;
        return Entry{x == x ? s.off[b] + static_cast<double>(x) : -INFINITY, place_of(b, id + 1)};
    };
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < n_segs * kSeg; i += kPickThreads) list(value(s.chosen, i));
    __syncthreads();
    count = s.count;
    Entry mine{-INFINITY, 0};
    if (count <= kListMax) {
        rank_list(s, count, p.width);
        if (static_cast<int>(threadIdx.x) < min(count, p.width)) mine = s.chosen[threadIdx.x];
    } else {
        Entry * segs = s.list;                             // chosen takes the values
        if (static_cast<int>(threadIdx.x) < n_segs) segs[threadIdx.x] = s.chosen[threadIdx.x];
        __syncthreads();
        one_by_one(s, p.width, n_segs * kSeg, [&](int i) { return value(segs, i); });
        if (static_cast<int>(threadIdx.x) < p.width) mine = s.chosen[threadIdx.x];
    }
    if (static_cast<int>(threadIdx.x) >= p.width) return;
    const int out = row0 + threadIdx.x;
    if (static_cast<int>(threadIdx.x) >= count) {
        p.parents[out] = out;
        p.tokens[out] = -1;
        p.scores_out[out] = -INFINITY;
        p.done_out[out] = 1;
        return;
    }
    const int id = static_cast<int>(static_cast<uint32_t>(mine.at)) - 1;
    int ended = id < 0;
    for (int k = 0; k < p.n_stop; ++k) ended |= p.stop_ids[k] == id;
    p.parents[out] = row0 + static_cast<int>(mine.at >> 32);
    p.tokens[out] = id;
    p.scores_out[out] = static_cast<float>(mine.score);
    p.done_out[out] = ended;
}

struct BeamPlan {
    int n_units, n_segs;
    size_t units_bytes, bytes;
};

BeamPlan beam_plan(int64_t rows, int32_t vocab) {
    BeamPlan pl{};
    pl.n_units = (vocab + kLoads * 256 - 1) / (kLoads * 256);
    pl.n_segs = (vocab + kSeg - 1) / kSeg;
    pl.units_bytes = static_cast<size_t>(rows) * pl.n_units * sizeof(Unit);
    pl.bytes = pl.units_bytes + (static_cast<size_t>(rows) * pl.n_segs * sizeof(float) + 15) / 16 * 16;
    return pl;
}

int check_beams(int32_t n_groups, int32_t width, int32_t vocab, const char * who) {
    if (width < 1 || width > kMaxWidth) return fail(QA_ERR_INVALID, std::string(who) + ": 1 to 64 beams");
    if (n_groups < 0 || static_cast<int64_t>(n_groups) * width > 65535) return fail(QA_ERR_INVALID, std::string(who) + ": at most 65535 rows");
    if (vocab < width || vocab > kMaxCapacity) return fail(QA_ERR_INVALID, std::string(who) + ": vocabulary out of range");
    return QA_OK;
}

struct ReorderParams {
    int32_t * refs;
    int32_t * tables;
    const int32_t * rows;
    const int32_t * parents;
    const int32_t * lens;
    int32_t * ids;
    const int32_t * tokens;
    const int32_t * ids_len;
    int32_t n_pages, n_rows, stride, shift, n, ids_stride, table_blocks;
};

constexpr int kMaxBeams = 1024, kCols = 8, kReorderThreads = 256;

// A workgroup per 8 columns of the tables or of the ids, with all rows: what the rows hold is read into LDS, and then each entry
// is written by one thread.  Only counts of entries that change are touched.  Its time is dependent loads: 2.3 us for 4 beams, 5.0 for 64.
__global__ __launch_bounds__(kReorderThreads) void beam_reorder_kernel(ReorderParams p) {
    __shared__ __attribute__((aligned(16))) int s_row[kMaxBeams];
    __shared__ int s_old[kMaxBeams * kCols];
    const bool pages = static_cast<int>(blockIdx.x) < p.table_blocks;
    int32_t * data = pages ? p.tables : p.ids;
    const int stride = pages ? p.stride : p.ids_stride;
    const int col0 = (static_cast<int>(blockIdx.x) - (pages ? 0 : p.table_blocks)) * kCols;
    for (int i = threadIdx.x; i < p.n; i += kReorderThreads) {
        const int row = p.rows ? p.rows[i] : i;
        s_row[i] = row >= 0 && row < p.n_rows ? row : -1;
    }
    __syncthreads();
    if (p.rows) {                                          // a row listed before is left out
        bool again[kMaxBeams / kReorderThreads] = {};
#pragma unroll
        for (int u = 0; u < kMaxBeams / kReorderThreads; ++u) {
            const int i = threadIdx.x + u * kReorderThreads;
            if (i >= p.n) continue;
            const int row = s_row[i];
            int hits = 0;
#pragma unroll 4
            for (int k = 0; k < i; k += 4) {               // four per LDS read, reads in flight together
                const i4 v = *reinterpret_cast<const i4 *>(s_row + k);
#pragma unroll
                for (int w = 0; w < 4; ++w) hits += k + w < i && v[w] == row;
            }
            again[u] = hits > 0;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMaxBeams / kReorderThreads; ++u) {
            const int i = threadIdx.x + u * kReorderThreads;
            if (i < p.n && again[u]) s_row[i] = -1;
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < p.n * kCols; e += kReorderThreads) {
        const int i = e / kCols, col = col0 + e % kCols;
        s_old[e] = s_row[i] >= 0 && col < stride ? data[static_cast<int64_t>(s_row[i]) * stride + col] : -1;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.n * kCols; e += kReorderThreads) {
        const int i = e / kCols, col = col0 + e % kCols, from = p.parents[i];
        if (s_row[i] < 0 || col >= stride || from < 0 || from >= p.n || s_row[from] < 0) continue;
        int32_t * to = data + static_cast<int64_t>(s_row[i]) * stride + col;
        const int old = s_old[e];
        int now = s_old[from * kCols + e % kCols];
        if (!pages) {
            if (p.tokens && col == p.ids_len[i] && p.tokens[i] >= 0) now = p.tokens[i];
            if (now != old) *to = now;
            continue;
        }
        const int len = p.lens[i];
        const int held = len <= 0 ? 0 : (len >> p.shift) + ((len & ((1 << p.shift) - 1)) != 0 ? 1 : 0);
        if (col >= held || now < 0 || now >= p.n_pages) now = -1;
        if (now == old) continue;
        *to = now;
        if (now >= 0) atomicAdd(&p.refs[now], 1);
        if (old >= 0 && old < p.n_pages) atomicSub(&p.refs[old], 1);
    }
}

}  // namespace
}  // namespace qa

extern "C" size_t qa_beam_select_workspace_bytes(int32_t n_groups, int32_t width, int32_t vocab) {
    using namespace qa;
    if (check_beams(n_groups, width, vocab, "qa_beam_select_workspace_bytes") != QA_OK) return 0;
    return beam_plan(static_cast<int64_t>(n_groups) * width, vocab).bytes;
}

extern "C" int qa_beam_select(const float * logits, int32_t n_groups, int32_t width, int32_t vocab, const float * scores,
                              const int32_t * done, const int32_t * stop_ids, int32_t n_stop, int32_t * parents, int32_t * tokens,
                              float * scores_out, int32_t * done_out, void * workspace, size_t workspace_bytes, void * stream) {
    using namespace qa;
    const char * who = "qa_beam_select";
    if (check_beams(n_groups, width, vocab, who) != QA_OK) return QA_ERR_INVALID;
    if (n_stop < 0 || n_stop > kMaxStops) return fail(QA_ERR_INVALID, "qa_beam_select: 0 to 64 stop ids");
    if (n_groups == 0) return QA_OK;
    if (!logits || !scores || !parents || !tokens || !scores_out || !done_out || (n_stop > 0 && !stop_ids)) {
        return fail(QA_ERR_INVALID, "qa_beam_select: null pointer");
    }
    const int rows = n_groups * width;
    const BeamPlan pl = beam_plan(rows, vocab);
    if (!workspace || workspace_bytes < pl.bytes) return fail(QA_ERR_INVALID, "qa_beam_select: workspace too small (qa_beam_select_workspace_bytes)");
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return fail(QA_ERR_INVALID, "qa_beam_select: workspace must be aligned to 16 bytes");
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    BeamParams p{};
    p.logits = logits;
    p.scores = scores;
    p.done = done;
    p.stop_ids = stop_ids;
    p.parents = parents;
    p.tokens = tokens;
    p.scores_out = scores_out;
    p.done_out = done_out;
    p.units = static_cast<Unit *>(workspace);
    p.seg_max = reinterpret_cast<float *>(static_cast<char *>(workspace) + pl.units_bytes);
    p.width = width;
    p.vocab = vocab;
    p.n_stop = n_stop;
    p.n_units = pl.n_units;
    p.n_segs = pl.n_segs;
    const dim3 grid(static_cast<unsigned>((pl.n_units + 3) / 4), static_cast<unsigned>(rows));
    hipLaunchKernelGGL(beam_units_kernel, grid, dim3(256), 0, as_stream(stream), p);
    QA_LAUNCH_CHECK("beam_units_kernel");
    hipLaunchKernelGGL(beam_pick_kernel, dim3(static_cast<unsigned>(n_groups)), dim3(kPickThreads), 0, as_stream(stream), p);
    QA_LAUNCH_CHECK("beam_pick_kernel");
    return QA_OK;
}

extern "C" int qa_beam_reorder(int32_t * refs, int32_t n_pages, int32_t * tables, int32_t n_rows, int32_t table_stride,
                               int32_t page_size, const int32_t * rows, const int32_t * parents, const int32_t * lens, int32_t n,
                               int32_t * ids, int32_t ids_stride, const int32_t * tokens, const int32_t * ids_len, void * stream) {
    using namespace qa;
    const char * who = "qa_beam_reorder";
    if (n < 0 || n > kMaxBeams) return fail(QA_ERR_INVALID, "qa_beam_reorder: 0 to 1024 beams");
    if (n_rows <= 0) return fail(QA_ERR_INVALID, "qa_beam_reorder: no rows");
    if ((refs != nullptr) != (tables != nullptr)) return fail(QA_ERR_INVALID, "qa_beam_reorder: null pointer");
    if (tables) {
        if (n_pages <= 0 || page_size < kPageMin || page_size > kPageMax || (page_size & (page_size - 1)) != 0) {
            return fail(QA_ERR_INVALID, "qa_beam_reorder: pages of 16, 32, 64, 128 or 256 positions");
        }
        if (check_table(n_rows, table_stride, page_size, who) != QA_OK) return QA_ERR_INVALID;
        if (n > 0 && !lens) return fail(QA_ERR_INVALID, "qa_beam_reorder: null pointer");
    }
    if (ids && (ids_stride <= 0 || ids_stride > kMaxCapacity)) return fail(QA_ERR_INVALID, "qa_beam_reorder: ids_stride out of range");
    if (n == 0 || (!tables && !ids)) return QA_OK;
    if (!parents || (ids && tokens && !ids_len)) return fail(QA_ERR_INVALID, "qa_beam_reorder: null pointer");
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    ReorderParams p{};
    p.refs = refs;
    p.tables = tables;
    p.rows = rows;
    p.parents = parents;
    p.lens = lens;
    p.ids = ids;
    p.tokens = tokens;
    p.ids_len = ids_len;
    p.n_pages = n_pages;
    p.n_rows = n_rows;
    p.stride = table_stride;
    p.shift = tables ? page_shift_of(page_size) : 0;
    p.n = n;
    p.ids_stride = ids_stride;
    p.table_blocks = tables ? (table_stride + kCols - 1) / kCols : 0;
    const int blocks = p.table_blocks + (ids ? (ids_stride + kCols - 1) / kCols : 0);
    hipLaunchKernelGGL(beam_reorder_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kReorderThreads), 0, as_stream(stream), p);
    QA_LAUNCH_CHECK("beam_reorder_kernel");
    return QA_OK;
}
