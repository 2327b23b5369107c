// Beam search: the best continuations over a group's beams and the vocabulary, and the beams' states put in their new order.
//
// Selection in two launches.  The first streams the logits once (a wave takes a unit of a row, values in registers): the largest
// value of every 64, and the unit's maximum and sum of exponentials.  The second, a workgroup per group, needs no more than
// those: a row's logarithm of its sum turns maxima into scores, and the new beams are among the values of the `width` best
// 64s, as any value outside has `width` better ones (of 64s that tie, the earlier has the lower ids).  It reads those again,
// width x 256 bytes.  Both of its choices, of 64s and of values, go the same way: a bound that at least `width` entries
// reach, a list of the entries that reach it, and each entry's rank in the list by counting.
// Exponentials are f32, sums and logarithms f64, and so are scores, so that candidates of different beams compare as in the formula.
#include "common.hpp"
#include "paged.hpp"
#include "wave.hpp"

#include <algorithm>

namespace qa {
namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // rows of an odd vocabulary start anywhere

constexpr int kSeg = 64;             // values per maximum
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
    int32_t n_rows, width, vocab, n_stop, n_units, n_segs;
};

// LOADS x 256 values per wave.
template <int LOADS>
__global__ __launch_bounds__(256) void beam_units_kernel(BeamParams p) {
    const int lane = threadIdx.x & (kWave - 1);
    const int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.y;
    if (unit >= p.n_units || (p.done && p.done[row] != 0)) return;       // a beam that is done has one candidate
    const float * x = p.logits + static_cast<int64_t>(row) * p.vocab;
    const int first = unit * LOADS * 256 + lane * 4;
    f4u v[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
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
    for (int u = 0; u < LOADS; ++u) {
        float seg = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[u][e] = v[u][e] == v[u][e] ? v[u][e] : -INFINITY;
            seg = fmaxf(seg, v[u][e]);
        }
        seg = fmaxf(seg, dpp_f<0xB1>(seg));
        seg = fmaxf(seg, dpp_f<0x4E>(seg));
        seg = fmaxf(seg, dpp_f<0x141>(seg));
        seg = fmaxf(seg, dpp_f<0x140>(seg));
        const int s = (unit * LOADS + u) * 4 + (lane >> 4);
        if ((lane & 15) == 0 && s < p.n_segs) p.seg_max[static_cast<int64_t>(row) * p.n_segs + s] = seg;
        most = fmaxf(most, seg);
    }
    most = wave_max_all(most);
    double sum = 0.0;
    if (most > -INFINITY) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += static_cast<double>(expf(v[u][e] - most));
        }
    }
    sum = wave_sum_d_all(sum);
    if (lane == 0) p.units[static_cast<int64_t>(row) * p.n_units + unit] = Unit{sum, most, 0.0f};
}

// A candidate: its score and its number in the order that settles ties.  -inf: none.
struct Entry {
    double score;
    int64_t at;
};
__device__ inline bool better(double a, int64_t i, double b, int64_t j) { return a > b || (a == b && i < j); }

__device__ inline double wave_best(double v, int64_t & at) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const double o = __shfl_xor(v, d, kWave);
        const int64_t i = __shfl_xor(at, d, kWave);
        if (better(o, i, v, at)) v = o, at = i;
    }
    return v;
}

struct PickLds {
    double off[kMaxWidth];           // what a row's values are raised by to become scores; -inf: none of them counts
    double stay[kMaxWidth];          // the score of a beam that is done
    Entry list[kListMax];
    Entry chosen[kMaxWidth];
    Entry wave[kPickWaves];
    int count, n_chosen;
};

// The `width` best of n entries, best first, into chosen.  score(i) is the i-th one's, which settles ties as well.
template <typename F>
__device__ inline void choose(PickLds & s, int width, int64_t n, F && score) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    // every wave's k-th best lane, k the same for all: at least k x waves >= width entries reach the least of them
    double best = -INFINITY;
    int64_t at = n;
    for (int64_t i = threadIdx.x; i < n; i += kPickThreads) {
        const double v = score(i);
        if (v > best) best = v, at = i;
    }
    double bound = best;
    int64_t bound_at = at;
    for (int k = (width + kPickWaves - 1) / kPickWaves; k > 0; --k) {
        double v = best;
        int64_t i = at;
        v = wave_best(v, i);
        bound = v;
        bound_at = i;
        if (best == v && at == i) best = -INFINITY, at = n;
    }
    if (threadIdx.x == 0) s.count = 0, s.n_chosen = 0;
    if (lane == 0) s.wave[wave] = Entry{bound, bound_at};
    __syncthreads();
    for (int w = 0; w < kPickWaves; ++w) {
        if (better(bound, bound_at, s.wave[w].score, s.wave[w].at)) bound = s.wave[w].score, bound_at = s.wave[w].at;
    }
    for (int64_t i = threadIdx.x; i < n; i += kPickThreads) {
        const double v = score(i);
        if (!(v > -INFINITY) || better(bound, bound_at, v, i)) continue;
        const int to = atomicAdd(&s.count, 1);
        if (to < kListMax) s.list[to] = Entry{v, i};
    }
    __syncthreads();
    const int count = s.count;
    if (count <= kListMax) {
        if (static_cast<int>(threadIdx.x) < count) {
            const Entry e = s.list[threadIdx.x];
            int rank = 0;
            for (int k = 0; k < count; ++k) rank += better(s.list[k].score, s.list[k].at, e.score, e.at);
            if (rank < width) s.chosen[rank] = e;
        }
        if (threadIdx.x == 0) s.n_chosen = min(count, width);
        __syncthreads();
        return;
    }
    // one by one, each the best of those behind the one before
    Entry last{INFINITY, -1};
    for (int r = 0; r < width; ++r) {
        double v = -INFINITY;
        int64_t a = n;
        for (int64_t i = threadIdx.x; i < n; i += kPickThreads) {
            const double x = score(i);
            if (x > -INFINITY && better(last.score, last.at, x, i) && better(x, i, v, a)) v = x, a = i;
        }
        v = wave_best(v, a);
        __syncthreads();
        if (lane == 0) s.wave[wave] = Entry{v, a};
        __syncthreads();
        last = s.wave[0];
        for (int w = 1; w < kPickWaves; ++w) {
            if (better(s.wave[w].score, s.wave[w].at, last.score, last.at)) last = s.wave[w];
        }
        if (threadIdx.x == 0) s.chosen[r] = last;
    }
    if (threadIdx.x == 0) s.n_chosen = width;              // more than kListMax entries count
    __syncthreads();
}

__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(BeamParams p) {
    __shared__ PickLds s;
    __shared__ Entry s_segs[kMaxWidth];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    const int row0 = blockIdx.x * p.width;
    for (int b = wave; b < p.width; b += kPickWaves) {
        const int row = row0 + b;
        const double score = static_cast<double>(p.scores[row]);
        const bool counts = score > -INFINITY && score < INFINITY, done = p.done && p.done[row] != 0;
        double off = -INFINITY;
        if (counts && !done) {
            const Unit * units = p.units + static_cast<int64_t>(row) * p.n_units;
            float most = -INFINITY;
            for (int u = lane; u < p.n_units; u += kWave) most = fmaxf(most, units[u].most);
            most = wave_max_all(most);
            double sum = 0.0;
            for (int u = lane; u < p.n_units; u += kWave) {
                if (units[u].most > -INFINITY) sum += units[u].sum * exp(static_cast<double>(units[u].most) - most);
            }
            sum = wave_sum_d_all(sum);
            if (most > -INFINITY && most < INFINITY) off = score - (log(sum) + most);
        }
        if (lane == 0) {
            s.off[b] = off;
            s.stay[b] = counts && done ? score : -INFINITY;
        }
    }
    __syncthreads();
    // entries of a beam: itself, where it is done, and its 64s
    const int per_beam = p.n_segs + 1;
    choose(s, p.width, static_cast<int64_t>(p.width) * per_beam, [&](int64_t i) {
        const int b = static_cast<int>(i / per_beam), seg = static_cast<int>(i - static_cast<int64_t>(b) * per_beam) - 1;
        if (seg < 0) return s.stay[b];
        const double off = s.off[b];
        return off > -INFINITY ? off + static_cast<double>(p.seg_max[static_cast<int64_t>(row0 + b) * p.n_segs + seg]) : -INFINITY;
    });
    const int n_segs = s.n_chosen;
    if (static_cast<int>(threadIdx.x) < n_segs) s_segs[threadIdx.x] = s.chosen[threadIdx.x];
    __syncthreads();
    // put in order of beam and place, so that an entry's number settles ties
    if (static_cast<int>(threadIdx.x) < n_segs) {
        const Entry e = s_segs[threadIdx.x];
        int rank = 0;
        for (int k = 0; k < n_segs; ++k) rank += s_segs[k].at < e.at;
        s.chosen[rank] = e;
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < n_segs) s_segs[threadIdx.x] = s.chosen[threadIdx.x];
    __syncthreads();
    auto place = [&](int64_t i, int & b, int & id) {       // of value i % 64 of the chosen 64
        const int64_t at = s_segs[i / kSeg].at;
        b = static_cast<int>(at / per_beam);
        const int seg = static_cast<int>(at - static_cast<int64_t>(b) * per_beam) - 1;
        id = seg < 0 ? -1 : seg * kSeg + static_cast<int>(i % kSeg);
        return seg < 0 ? i % kSeg == 0 : id < p.vocab;
    };
    choose(s, p.width, static_cast<int64_t>(n_segs) * kSeg, [&](int64_t i) {
        int b, id;
        if (!place(i, b, id)) return static_cast<double>(-INFINITY);
        if (id < 0) return s.stay[b];
        const float x = p.logits[static_cast<int64_t>(row0 + b) * p.vocab + id];
        return x == x ? s.off[b] + static_cast<double>(x) : -INFINITY;
    });
    if (static_cast<int>(threadIdx.x) >= p.width) return;
    const int r = threadIdx.x, out = row0 + r;
    if (r >= s.n_chosen) {
        p.parents[out] = out;
        p.tokens[out] = -1;
        p.scores_out[out] = -INFINITY;
        p.done_out[out] = 1;
        return;
    }
    int b, id;
    place(s.chosen[r].at, b, id);
    int ended = id < 0;
    for (int k = 0; k < p.n_stop; ++k) ended |= p.stop_ids[k] == id;
    p.parents[out] = row0 + b;
    p.tokens[out] = id;
    p.scores_out[out] = static_cast<float>(s.chosen[r].score);
    p.done_out[out] = ended;
}

// How the first launch cuts rows: short units where they are what fills the GPU.
struct BeamPlan {
    int loads, n_units, n_segs;
    size_t units_bytes, bytes;
};

BeamPlan beam_plan(int64_t rows, int32_t vocab) {
    BeamPlan pl{};
    pl.loads = rows * vocab > (int64_t{1} << 22) ? 8 : 2;
    pl.n_units = (vocab + pl.loads * 256 - 1) / (pl.loads * 256);
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
// is written by one thread.  Only counts of entries that change are touched.
__global__ __launch_bounds__(kReorderThreads) void beam_reorder_kernel(ReorderParams p) {
    __shared__ int s_row[kMaxBeams], s_old[kMaxBeams * kCols];
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
            for (int k = 0; k < i; ++k) again[u] = again[u] || s_row[k] == s_row[i];
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
    p.n_rows = rows;
    p.width = width;
    p.vocab = vocab;
    p.n_stop = n_stop;
    p.n_units = pl.n_units;
    p.n_segs = pl.n_segs;
    const dim3 grid(static_cast<unsigned>((pl.n_units + 3) / 4), static_cast<unsigned>(rows));
    const auto kernel = pl.loads == 8 ? &beam_units_kernel<8> : &beam_units_kernel<2>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, as_stream(stream), p);
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
