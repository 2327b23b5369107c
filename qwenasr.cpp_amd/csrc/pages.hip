// Bookkeeping of a paged K/V cache on the device: pages given, shared, taken back, copied and moved together.
//
// The counts and tables are a few KB, so one workgroup plans a call (who needs what, which pages are free) and what it
// costs is its dependent loads; pages themselves are 0.4 to 57 MB over all layers, so they are copied by a grid of their
// own behind the plan, 16 KB per workgroup, bound by HBM.  The plan reaches the copies through the workspace: nothing
// waits inside a kernel and the host reads nothing.  Every choice is by lowest number in list order, and counts change by
// integer atomics only, so results do not depend on timing.
#include "common.hpp"
#include "paged.hpp"

#include <algorithm>

namespace qa {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));

constexpr int kMaxList = 1024;       // rows or pairs of one call: one thread each in the plan
constexpr int kPlanThreads = 1024;
constexpr int kScan = 8;             // counts per thread and pass over them
constexpr int kPieceBytes = 16384;   // of a page, per workgroup
constexpr int kCopyThreads = 256;

// int32 workspace: [0] the pairs to copy, then the lists
constexpr int kWsHead = 16;

// Pairs of an extend: one per list entry, and behind them, where dst says so, one per page given.
constexpr int kBehind = -2;
__host__ __device__ inline int64_t extend_pairs(int n_pages) { return static_cast<int64_t>(kMaxList) + n_pages; }

__device__ inline bool is_page(int page, int n_pages) { return page >= 0 && page < n_pages; }
__host__ __device__ inline int pages_of_positions(int n, int shift) {
    return n <= 0 ? 0 : (n >> shift) + ((n & ((1 << shift) - 1)) != 0 ? 1 : 0);
}

// Exclusive prefix sum of v over the workgroup's threads; *total gets the sum.  part: one slot per wave.
template <typename T>
__device__ inline T block_scan(T v, T * part, T * total) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    T sum = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const T o = __shfl_up(sum, d, kWave);
        if (lane >= d) sum += o;
    }
    __syncthreads();                 // part may still be read from the scan before
    if (lane == kWave - 1) part[wave] = sum;
    __syncthreads();
    T before = 0, all = 0;
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
        if (w < wave) before += part[w];
        all += part[w];
    }
    *total = all;
    return before + sum - v;
}

struct ExtendParams {
    int32_t * refs;
    int32_t * tables;
    const int32_t * rows;
    const int32_t * n_past;
    const int32_t * n_new;
    int32_t * missing;
    int32_t * ws;
    int32_t n_pages, n_rows, stride, shift, n;
};

// Thread i < n plans list entry i.  The kernel's time is its dependent loads, so each is made for all entries at once: up to
// kSpan table entries per list entry (a decode step's one or two) by the entry's thread, longer spans by a wave each; the
// counts of the first pages are read before anything is known.
// A page that others hold is as a rule the first one written: a beam goes on behind what it shares.  Who copies it is found in
// LDS.  Only where a sequence has gone back, and is about to write pages behind its first that others hold, all entries
// are counted per page in the workspace (`spread`).  Traced, 32 rows behind 3913 positions: 6.4 us where nothing is shared, 9.2 with one
// shared page each, 17.2 and 18.0 where each has gone back over 4 and 10 shared pages.
constexpr int kSpan = 4;

__global__ __launch_bounds__(kPlanThreads) void pages_extend_kernel(ExtendParams p) {
    __shared__ __attribute__((aligned(16))) int s_row[kMaxList], s_claim[kMaxList];
    __shared__ int s_j0[kMaxList], s_j1[kMaxList];
    __shared__ int s_need[kMaxList];
    __shared__ long long s_base[kMaxList], s_part[kPlanThreads / kWave];
    __shared__ int s_behind;
    const int i = threadIdx.x, lane = i & (kWave - 1), wave = i >> 6;
    int32_t * src = p.ws + kWsHead;
    int32_t * dst = src + extend_pairs(p.n_pages);
    int32_t * list = dst + extend_pairs(p.n_pages);   // the free pages that are given, lowest first
    int32_t * spare = list + p.n_pages;       // spread: listed entries that hold a page, less all that do
    int32_t * last = spare + p.n_pages;       // and the last list entry among them
    // free pages among kScan counts, as a mask
    auto free_mask = [&](int64_t at) {
        unsigned mask = 0;
#pragma unroll
        for (int u = 0; u < kScan; ++u) {
            if (at + u < p.n_pages && p.refs[at + u] <= 0) mask |= 1u << u;
        }
        return mask;
    };
    unsigned mask = free_mask(static_cast<int64_t>(i) * kScan);
    int row = -1, j0 = 0, j1 = 0, claim = -1;
    if (i < p.n) {
        row = p.rows ? p.rows[i] : i;
        if (row < 0 || row >= p.n_rows) row = -1;
        const int past = p.n_past[i], add = min(p.n_new[i], kMaxCapacity - 1);
        if (past < 0 || past > kMaxCapacity || add <= 0) row = -1;
        if (row >= 0) {
            j1 = min(p.stride, pages_of_positions(past + add, p.shift));
            j0 = min(past >> p.shift, j1);
        }
    }
    if (i == 0) s_behind = 0;
    const bool wide = __syncthreads_or(j1 - j0 > kSpan);
    s_row[i] = row;
    int32_t * table = p.tables + static_cast<int64_t>(max(row, 0)) * p.stride;
    int entry[kSpan];
#pragma unroll
    for (int k = 0; k < kSpan; ++k) entry[k] = j0 + k < j1 ? table[j0 + k] : 0;
    __syncthreads();
    // entries ahead in the list, four per LDS read and whole reads in flight together (row by row 32 entries took 1 us more)
    const int ahead = min(i, p.n);
    auto count_ahead = [&](const int * list, int value) {
        int hits = 0;
#pragma unroll 4
        for (int k = 0; k < ahead; k += 4) {
            const i4 v = *reinterpret_cast<const i4 *>(list + k);
#pragma unroll
            for (int u = 0; u < 4; ++u) hits += k + u < ahead && v[u] == value;
        }
        return hits;
    };
    if (count_ahead(s_row, row) > 0) row = -1, j0 = j1 = 0;   // listed before
    int held[kSpan];
#pragma unroll
    for (int k = 0; k < kSpan; ++k) held[k] = j0 + k < j1 && is_page(entry[k], p.n_pages) ? p.refs[entry[k]] : 0;
    const int holders = held[0];
    if (holders > 1) claim = entry[0];
    bool behind = false;
#pragma unroll
    for (int k = 1; k < kSpan; ++k) behind = behind || held[k] > 1;
    s_claim[i] = claim;
    if (__any(behind) && lane == 0) s_behind = 1;
    __syncthreads();
    bool spread = s_behind != 0;
    if (claim >= 0) {
        if (holders - count_ahead(s_claim, claim) <= 1) claim = -1;   // those ahead take a copy, the last holder keeps the page
    }
    int need = claim >= 0 ? 1 : 0;
    if (!wide) {
#pragma unroll
        for (int k = 0; k < kSpan; ++k) need += j0 + k < j1 && !is_page(entry[k], p.n_pages);
    }
    __syncthreads();
    s_claim[i] = claim;
    s_row[i] = row;
    s_j0[i] = j0;
    s_j1[i] = j1;
    s_need[i] = need;
    // every entry that list entry s writes, a wave per list entry and 64 entries at a time
    auto walk = [&](auto && each, auto && done) {
        for (int s = wave; s < p.n; s += kPlanThreads / kWave) {
            const int32_t * of = p.tables + static_cast<int64_t>(max(s_row[s], 0)) * p.stride;
            for (int b = s_j0[s]; b < s_j1[s]; b += kWave) {
                const int j = b + lane, page = of[min(j, s_j1[s] - 1)];
                each(s, j, j < s_j1[s], page);
            }
            done(s);
        }
        __syncthreads();
    };
    const auto nothing = [](int) {};
    // of the listed entries that hold a page the last one keeps it, unless others hold it; read past the caches, behind atomics
    auto copied = [&](int s, int page) {
        const int n = __hip_atomic_load(&spare[page], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return n < 0 || (n == 0 && __hip_atomic_load(&last[page], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != s);
    };
    int count = 0;
    auto add_need = [&](int s) {
        if (lane == 0) s_need[s] += count;
        count = 0;
    };
    if (wide || spread) __syncthreads();
    if (wide) {
        walk([&](int s, int j, bool in, int page) {
            const bool there = is_page(page, p.n_pages);
            count += __popcll(__ballot(in && !there));
            behind = behind || (in && j > s_j0[s] && there && p.refs[page] > 1);
        }, add_need);
        spread = __syncthreads_or(behind);
    }
    if (spread) {
        walk([&](int, int, bool in, int page) {
            if (!in || !is_page(page, p.n_pages)) return;
            spare[page] = -p.refs[page];
            last[page] = -1;
        }, nothing);
        walk([&](int s, int, bool in, int page) {
            if (!in || !is_page(page, p.n_pages)) return;
            atomicAdd(&spare[page], 1);
            atomicMax(&last[page], s);
        }, nothing);
        claim = -1;
        s_claim[i] = -1;
        s_need[i] = 0;
        __syncthreads();
        walk([&](int s, int, bool in, int page) {
            count += __popcll(__ballot(in && (!is_page(page, p.n_pages) || copied(s, page))));
        }, add_need);
    }
    long long total = 0;
    const long long base = block_scan<long long>(i < p.n ? s_need[i] : 0, s_part, &total);
    s_base[i] = base;
    // free pages, lowest first, until there are enough (or none left: then the count tells what is lacking)
    long long found = 0;
    for (int64_t b = 0; b < p.n_pages && found < total; b += kPlanThreads * kScan) {
        const int64_t at = b + static_cast<int64_t>(i) * kScan;
        if (b > 0) mask = free_mask(at);
        long long here = 0;
        long long r = found + block_scan<long long>(__popc(mask), s_part, &here);
        for (; mask != 0 && r < total; mask &= mask - 1, ++r) list[r] = static_cast<int32_t>(at + __ffs(mask) - 1);
        found += here;
    }
    if (i == 0) *p.missing = total <= found ? 0 : static_cast<int32_t>(min(total - found, static_cast<long long>(INT32_MAX)));
    if (i < p.n && (total > found || claim < 0)) dst[i] = spread && total <= found ? kBehind : -1;   // nothing to copy for this entry
    if (total > found) return;                            // nothing is changed
    if (spread && i == 0) p.ws[0] = static_cast<int32_t>(p.n + total);
    __syncthreads();
    if (i < p.n && need > 0 && claim >= 0) {
        const int page = list[base];
        src[i] = claim;
        dst[i] = page;
        table[j0] = page;
        p.refs[page] = 1;
        atomicSub(&p.refs[claim], 1);
    }
    if (!wide && !spread) {
        long long at = base + (claim >= 0 ? 1 : 0);
#pragma unroll
        for (int k = 0; k < kSpan; ++k) {
            if (j0 + k >= j1 || is_page(entry[k], p.n_pages)) continue;
            const int page = list[at++];
            table[j0 + k] = page;
            p.refs[page] = 1;
        }
        return;
    }
    for (int s = wave; s < p.n; s += kPlanThreads / kWave) {
        if (s_need[s] == 0) continue;
        int32_t * of = p.tables + static_cast<int64_t>(s_row[s]) * p.stride;
        long long at = s_base[s] + (s_claim[s] >= 0 ? 1 : 0);
        // the first entry of a claim holds a page and is passed over here, whether its new number is visible yet or not
        for (int b = s_j0[s]; b < s_j1[s]; b += kWave) {
            const int j = b + lane, old = of[min(j, s_j1[s] - 1)];
            const bool in = j < s_j1[s], none = !is_page(old, p.n_pages);
            const bool copy = spread && in && !none && copied(s, old);
            const bool want = (in && none) || copy;
            const uint64_t all = __ballot(want);
            if (want) {
                const long long r = at + __popcll(all & ((1ull << lane) - 1));
                const int page = list[r];
                of[j] = page;
                p.refs[page] = 1;
                if (spread) {
                    src[p.n + r] = old;
                    dst[p.n + r] = copy ? page : -1;
                }
                if (copy) atomicSub(&p.refs[old], 1);
            }
            at += __popcll(all);
        }
    }
}

// A pair whose dst a later pair has too, or that some pair reads, is left out (threads check one pair each).
__device__ inline bool pair_stands(const int32_t * src, const int32_t * dst, int i, int n) {
    const int d = dst[i];
    int clash = 0;
    for (int k = threadIdx.x; k < n; k += blockDim.x) clash |= (k > i && dst[k] == d) || src[k] == d;
    return !__syncthreads_or(clash);
}

__global__ __launch_bounds__(256) void pages_fork_kernel(int32_t * refs, int n_pages, int32_t * tables, int n_rows, int stride,
                                                         int shift, const int32_t * src, const int32_t * dst,
                                                         const int32_t * len, int n) {
    const int i = blockIdx.x;
    if (!pair_stands(src, dst, i, n)) return;
    const int a = src[i], b = dst[i];
    if (a < 0 || a >= n_rows || b < 0 || b >= n_rows) return;
    const int held = pages_of_positions(len[i], shift);
    const int32_t * from = tables + static_cast<int64_t>(a) * stride;
    int32_t * to = tables + static_cast<int64_t>(b) * stride;
    for (int j = threadIdx.x; j < stride; j += blockDim.x) {
        const int old = to[j];
        int page = j < held ? from[j] : -1;
        if (!is_page(page, n_pages)) page = -1;
        to[j] = page;
        if (page >= 0) atomicAdd(&refs[page], 1);
        if (is_page(old, n_pages)) atomicSub(&refs[old], 1);
    }
}

// The exchange hands each entry's page to one thread, also where a row is listed twice.
__global__ __launch_bounds__(256) void pages_free_kernel(int32_t * refs, int n_pages, int32_t * tables, int n_rows, int stride,
                                                         int shift, const int32_t * rows, const int32_t * keep) {
    const int row = rows[blockIdx.x];
    if (row < 0 || row >= n_rows) return;
    int32_t * table = tables + static_cast<int64_t>(row) * stride;
    for (int j = (keep ? pages_of_positions(keep[blockIdx.x], shift) : 0) + static_cast<int>(threadIdx.x); j < stride; j += blockDim.x) {
        const int old = atomicExch(&table[j], -1);
        if (is_page(old, n_pages)) atomicSub(&refs[old], 1);
    }
}

struct CopyParams {
    char * pages;
    const int32_t * src;
    const int32_t * dst;
    const int32_t * count;   // pairs that the device has counted, or null
    int64_t page_bytes;      // one (layer, K or V) block of a page
    int32_t n_pages, n, check;
};

// Workgroup (piece of the block, (layer, K or V), pair): 16 bytes per lane, 4 loads in flight, whole lines.
// ONCE: past the caches.  A compaction reads every page once: 24 sequences' 823 MB 165 instead of 174 us.  Copies of one parent's
// page find it in the caches: 32 of them 31 us with the plan, 38 past the caches.
template <bool ONCE>
__global__ __launch_bounds__(kCopyThreads) void pages_copy_kernel(CopyParams p) {
    int n = ONCE ? min(*p.count, p.n) : p.n;
    for (int i = blockIdx.z; i < n; i += gridDim.z) {
        if (p.check && !pair_stands(p.src, p.dst, i, n)) continue;   // uniform for the workgroup
        const int a = p.src[i], b = p.dst[i];
        if (!ONCE && p.count && b == kBehind) n = *p.count;   // read only then: an extend's usual copies wait for nothing else
        if (!is_page(a, p.n_pages) || !is_page(b, p.n_pages) || a == b) continue;
        const int64_t block = static_cast<int64_t>(blockIdx.y) * p.n_pages;
        const int64_t at = static_cast<int64_t>(blockIdx.x) * kPieceBytes + threadIdx.x * 16;
        const u4 * from = reinterpret_cast<const u4 *>(p.pages + (block + a) * p.page_bytes + at);
        u4 * to = reinterpret_cast<u4 *>(p.pages + (block + b) * p.page_bytes + at);
        constexpr int kPer = kPieceBytes / (kCopyThreads * 16);
        u4 v[kPer];
        const int64_t left = p.page_bytes - at;           // a block is at least 4 KB and may end inside a piece
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            if (left <= u * kCopyThreads * 16) continue;
            if constexpr (ONCE) v[u] = __builtin_nontemporal_load(from + u * kCopyThreads);
            else v[u] = from[u * kCopyThreads];
        }
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            if (left <= u * kCopyThreads * 16) continue;
            if constexpr (ONCE) __builtin_nontemporal_store(v[u], to + u * kCopyThreads);
            else to[u * kCopyThreads] = v[u];
        }
    }
}

// Live pages, then the free numbers before that count and the live ones behind it, each lowest first, and every page's
// place after the move.
__global__ __launch_bounds__(kPlanThreads) void pages_compact_plan_kernel(const int32_t * refs, int n_pages, int32_t * ws, int32_t * n_live) {
    __shared__ int s_part[kPlanThreads / kWave];
    int32_t * place = ws + kWsHead;
    int32_t * holes = place + n_pages;
    int32_t * movers = holes + n_pages;
    const int i = threadIdx.x;
    int live = 0;
    for (int64_t b = 0; b < n_pages; b += kPlanThreads * kScan) {
        const int64_t at = b + static_cast<int64_t>(i) * kScan;
        int c = 0, here = 0;
#pragma unroll
        for (int u = 0; u < kScan; ++u) c += at + u < n_pages && refs[at + u] > 0;
        block_scan<int>(c, s_part, &here);
        live += here;
    }
    int n_holes = 0, n_movers = 0;
    for (int64_t b = 0; b < n_pages; b += kPlanThreads * kScan) {
        const int64_t at = b + static_cast<int64_t>(i) * kScan;
        unsigned used = 0, there = 0, behind = 0;
#pragma unroll
        for (int u = 0; u < kScan; ++u) {
            if (at + u >= n_pages) continue;
            there |= 1u << u;
            if (refs[at + u] > 0) used |= 1u << u;
            if (at + u >= live) behind |= 1u << u;
        }
        const unsigned hole = there & ~used & ~behind, mover = used & behind;
        int here = 0;
        int r = n_holes + block_scan<int>(__popc(hole), s_part, &here);
        n_holes += here;
        for (unsigned m = hole; m != 0; m &= m - 1) holes[r++] = static_cast<int32_t>(at + __ffs(m) - 1);
        r = n_movers + block_scan<int>(__popc(mover), s_part, &here);
        n_movers += here;
        for (unsigned m = mover; m != 0; m &= m - 1) movers[r++] = static_cast<int32_t>(at + __ffs(m) - 1);
#pragma unroll
        for (int u = 0; u < kScan; ++u) {
            if (((there & ~mover) >> u) & 1) place[at + u] = (used >> u) & 1 ? static_cast<int32_t>(at + u) : -1;
        }
    }
    __syncthreads();
    for (int k = i; k < n_movers; k += kPlanThreads) place[movers[k]] = holes[k];
    if (i == 0) {
        ws[0] = n_movers;
        *n_live = live;
    }
}

// New numbers in the tables, counts at their pages' new places.  Page p's thread alone writes the counts of p and of the
// hole that it moves into, so refs_out may be refs.
__global__ __launch_bounds__(256) void pages_renumber_kernel(const int32_t * refs, const int32_t * tables, int32_t * refs_out,
                                                             int32_t * tables_out, const int32_t * ws, int n_pages,
                                                             int64_t entries) {
    const int32_t * place = ws + kWsHead;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x, first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int moved = ws[0];
    // the free numbers that are taken are the first ones: a page is one of them if it is free and before the last hole
    const int32_t * holes = place + n_pages;
    const int last_hole = moved > 0 ? holes[moved - 1] : -1;
    for (int64_t id = first; id < n_pages; id += step) {
        const int to = place[id];
        if (to < 0 && id <= last_hole) continue;          // its new page's thread writes it
        const int count = refs[id];
        if (to >= 0 && to != id) {
            refs_out[to] = count;
            refs_out[id] = 0;
        } else {
            refs_out[id] = count;
        }
    }
    for (int64_t e = first; e < entries; e += step) {
        const int page = tables[e];
        tables_out[e] = is_page(page, n_pages) ? place[page] : -1;
    }
}

int64_t block_bytes(const qa_kv_layout & l) {
    return static_cast<int64_t>(l.n_kv_heads) * l.max_seq * l.head_dim * static_cast<int64_t>(qa_kv_elem_bytes(l.cache_type));
}

int launch_copies(void * pages, const qa_kv_layout & l, const int32_t * src, const int32_t * dst, const int32_t * count, int32_t n,
                  int32_t most, bool once, bool check, hipStream_t stream) {
    CopyParams p{};
    p.pages = static_cast<char *>(pages);
    p.src = src;
    p.dst = dst;
    p.count = count;
    p.page_bytes = block_bytes(l);
    p.n_pages = l.n_streams;
    p.n = n;
    p.check = check ? 1 : 0;
    const dim3 grid(static_cast<unsigned>((p.page_bytes + kPieceBytes - 1) / kPieceBytes), static_cast<unsigned>(2 * l.n_layers),
                    static_cast<unsigned>(std::max(1, std::min(n, most))));
    const auto kernel = once ? &pages_copy_kernel<true> : &pages_copy_kernel<false>;
    hipLaunchKernelGGL(kernel, grid, dim3(kCopyThreads), 0, stream, p);
    QA_LAUNCH_CHECK("pages_copy_kernel");
    return QA_OK;
}

int check_list(int32_t n, const char * who) {
    if (n < 0 || n > kMaxList) return fail(QA_ERR_INVALID, std::string(who) + ": 0 to 1024 rows or pairs per call");
    return QA_OK;
}

int check_counts(const int32_t * refs, int32_t n_pages, const int32_t * tables, int32_t n_rows, int32_t stride, int32_t page_size,
                 const char * who) {
    if (n_pages <= 0 || page_size < kPageMin || page_size > kPageMax || (page_size & (page_size - 1)) != 0) {
        return fail(QA_ERR_INVALID, std::string(who) + ": pages of 16, 32, 64, 128 or 256 positions");
    }
    if (check_table(n_rows, stride, page_size, who) != QA_OK) return QA_ERR_INVALID;
    if (!refs || !tables) return fail(QA_ERR_INVALID, std::string(who) + ": null pointer");
    return QA_OK;
}

// The copies' grid has a layer's K and V in its second dimension and a row of a block in 16-byte lanes.
int check_pool(const void * pages, const qa_kv_layout * l, const char * who) {
    if (check_pages(l, who) != QA_OK) return QA_ERR_INVALID;
    if (!pages) return fail(QA_ERR_INVALID, std::string(who) + ": null pointer");
    if ((reinterpret_cast<uintptr_t>(pages) & 15) != 0) return fail(QA_ERR_INVALID, std::string(who) + ": pages must be aligned to 16 bytes");
    if (l->n_layers > 32767) return fail(QA_ERR_INVALID, std::string(who) + ": more than 32767 layers");
    return QA_OK;
}

}  // namespace
}  // namespace qa

extern "C" size_t qa_pages_workspace_bytes(const qa_kv_layout * layout) {
    using namespace qa;
    if (check_pages(layout, "qa_pages_workspace_bytes") != QA_OK) return 0;
    return (kWsHead + 2 * static_cast<size_t>(extend_pairs(layout->n_streams)) + 3 * static_cast<size_t>(layout->n_streams)) * sizeof(int32_t);
}

extern "C" int qa_pages_extend(void * pages, const qa_kv_layout * layout, int32_t * refs, int32_t * tables, int32_t n_rows,
                               int32_t table_stride, const int32_t * rows, const int32_t * n_past, const int32_t * n_new,
                               int32_t n, int32_t * missing, void * workspace, size_t workspace_bytes, void * stream) {
    using namespace qa;
    const char * who = "qa_pages_extend";
    if (check_pool(pages, layout, who) != QA_OK || check_list(n, who) != QA_OK) return QA_ERR_INVALID;
    if (check_counts(refs, layout->n_streams, tables, n_rows, table_stride, layout->max_seq, who) != QA_OK) return QA_ERR_INVALID;
    if (!missing || (n > 0 && (!n_past || !n_new))) return fail(QA_ERR_INVALID, "qa_pages_extend: null pointer");
    if (!workspace || workspace_bytes < qa_pages_workspace_bytes(layout)) {
        return fail(QA_ERR_INVALID, "qa_pages_extend: workspace too small (qa_pages_workspace_bytes)");
    }
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    ExtendParams p{};
    p.refs = refs;
    p.tables = tables;
    p.rows = rows;
    p.n_past = n_past;
    p.n_new = n_new;
    p.missing = missing;
    p.ws = static_cast<int32_t *>(workspace);
    p.n_pages = layout->n_streams;
    p.n_rows = n_rows;
    p.stride = table_stride;
    p.shift = page_shift_of(layout->max_seq);
    p.n = n;
    hipLaunchKernelGGL(pages_extend_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), p);
    QA_LAUNCH_CHECK("pages_extend_kernel");
    if (n == 0) return QA_OK;
    const int64_t pairs = extend_pairs(p.n_pages);
    return launch_copies(pages, *layout, p.ws + kWsHead, p.ws + kWsHead + pairs, p.ws, n, n, false, false, as_stream(stream));
}

extern "C" int qa_pages_fork(int32_t * refs, int32_t n_pages, int32_t * tables, int32_t n_rows, int32_t table_stride,
                             int32_t page_size, const int32_t * src, const int32_t * dst, const int32_t * len, int32_t n,
                             void * stream) {
    using namespace qa;
    const char * who = "qa_pages_fork";
    if (check_counts(refs, n_pages, tables, n_rows, table_stride, page_size, who) != QA_OK || check_list(n, who) != QA_OK) return QA_ERR_INVALID;
    if (n == 0) return QA_OK;
    if (!src || !dst || !len) return fail(QA_ERR_INVALID, "qa_pages_fork: null pointer");
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    hipLaunchKernelGGL(pages_fork_kernel, dim3(static_cast<unsigned>(n)), dim3(256), 0, as_stream(stream), refs, n_pages, tables, n_rows,
                       table_stride, page_shift_of(page_size), src, dst, len, n);
    QA_LAUNCH_CHECK("pages_fork_kernel");
    return QA_OK;
}

extern "C" int qa_pages_free(int32_t * refs, int32_t n_pages, int32_t * tables, int32_t n_rows, int32_t table_stride,
                             int32_t page_size, const int32_t * rows, const int32_t * keep, int32_t n, void * stream) {
    using namespace qa;
    const char * who = "qa_pages_free";
    if (check_counts(refs, n_pages, tables, n_rows, table_stride, page_size, who) != QA_OK || check_list(n, who) != QA_OK) return QA_ERR_INVALID;
    if (n == 0) return QA_OK;
    if (!rows) return fail(QA_ERR_INVALID, "qa_pages_free: null pointer");
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    hipLaunchKernelGGL(pages_free_kernel, dim3(static_cast<unsigned>(n)), dim3(256), 0, as_stream(stream), refs, n_pages, tables, n_rows,
                       table_stride, page_shift_of(page_size), rows, keep);
    QA_LAUNCH_CHECK("pages_free_kernel");
    return QA_OK;
}

extern "C" int qa_pages_copy(void * pages, const qa_kv_layout * layout, const int32_t * src, const int32_t * dst, int32_t n, void * stream) {
    using namespace qa;
    const char * who = "qa_pages_copy";
    if (check_pool(pages, layout, who) != QA_OK || check_list(n, who) != QA_OK) return QA_ERR_INVALID;
    if (n == 0) return QA_OK;
    if (!src || !dst) return fail(QA_ERR_INVALID, "qa_pages_copy: null pointer");
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    return launch_copies(pages, *layout, src, dst, nullptr, n, n, false, true, as_stream(stream));
}

extern "C" int qa_pages_compact(void * pages, const qa_kv_layout * layout, const int32_t * refs, const int32_t * tables, int32_t n_rows,
                                int32_t table_stride, int32_t * refs_out, int32_t * tables_out, int32_t * n_live, void * workspace,
                                size_t workspace_bytes, void * stream) {
    using namespace qa;
    const char * who = "qa_pages_compact";
    if (check_pool(pages, layout, who) != QA_OK) return QA_ERR_INVALID;
    if (check_counts(refs, layout->n_streams, tables, n_rows, table_stride, layout->max_seq, who) != QA_OK) return QA_ERR_INVALID;
    if (!refs_out || !tables_out || !n_live) return fail(QA_ERR_INVALID, "qa_pages_compact: null pointer");
    if (!workspace || workspace_bytes < qa_pages_workspace_bytes(layout)) {
        return fail(QA_ERR_INVALID, "qa_pages_compact: workspace too small (qa_pages_workspace_bytes)");
    }
    if (const int rc = check_stream(stream, who); rc != QA_OK) return rc;
    const int n_pages = layout->n_streams;
    int32_t * ws = static_cast<int32_t *>(workspace);
    hipLaunchKernelGGL(pages_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), refs, n_pages, ws, n_live);
    QA_LAUNCH_CHECK("pages_compact_plan_kernel");
    const int32_t * holes = ws + kWsHead + n_pages;
    if (n_pages > 1) {
        const int rc = launch_copies(pages, *layout, holes + n_pages, holes, ws, n_pages / 2, 256, true, false, as_stream(stream));
        if (rc != QA_OK) return rc;
    }
    const int64_t entries = static_cast<int64_t>(n_rows) * table_stride;
    const int64_t blocks = (std::max<int64_t>(entries, n_pages) + 255) / 256;
    hipLaunchKernelGGL(pages_renumber_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 1024))), dim3(256), 0, as_stream(stream),
                       refs, tables, refs_out, tables_out, ws, n_pages, entries);
    QA_LAUNCH_CHECK("pages_renumber_kernel");
    return QA_OK;
}
