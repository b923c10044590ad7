// The pages of a cache: rows appended to the pages of their sequences
// (pages_append), tables forked, freed and made longer (pages_fork), and rows of
// one page copied to another (pages_copy). Token t of a sequence is row t % page
// of page table[t / page].
//
// pages_append and pages_copy move K and V in one launch, whole float4s where rows
// allow it, with loads and stores past the L2, and are bound by memory: 4 x 4096 rows of 8
// heads of 128 to pages of 64 tokens by head, 268 MB in 47.5 us, 5.6 TB/s; 392 copies of 1 to
// 256 rows, 813 MB in 162 us, 5.0 TB/s (with half or twice the loads on their way, a quarter or
// four times the blocks, K and V by blocks of their own: 158 to 179). One row each of 64
// sequences, or 4 copies of 16 rows, take a launch, 3.4 us.
//
// pages_fork is three launches, because what a page is used for is known only once
// every sequence has said what it keeps, and which pages are free only after that:
//   1. a block for each sequence: its parent's pages into its new table, and what its
//      own old table's pages gain or lose into a sum for each page (integer atomics,
//      so their order changes nothing);
//   2. uses and sums into new uses, 1024 pages a block, which counts its free ones;
//      one block more sums up what the sequences ask for;
//   3. the free pages in order of their numbers to the sequences in theirs.
// 512 sequences with tables of 2048 entries and 394 k pages: 17.6, 4.7 and 7.6 us; 8 us of
// the first are its atomics, the rest loads that wait for one another.
// The sums are zeros before and after a call. Few sequences over few pages take one launch.
#include "kernels.hpp"
#include "whole.hpp"

namespace jade {
namespace hipk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr uint32_t kBlockWords = 2 * kThreads;  // elements (float4s, or floats) of each tensor that a block moves
constexpr uint32_t kMaxBlocks = 1u << 20;

__device__ inline bool is_whole(float x, uint32_t most) { return x >= 0.f && x < float(most) && x == truncf(x); }

template <typename T>
__device__ inline void move(const float *k, const float *v, size_t from, float *k_to, float *v_to, size_t to) {
    const T x = __builtin_nontemporal_load(reinterpret_cast<const T *>(k) + from);
    const T y = __builtin_nontemporal_load(reinterpret_cast<const T *>(v) + from);
    __builtin_nontemporal_store(x, reinterpret_cast<T *>(k_to) + to);
    __builtin_nontemporal_store(y, reinterpret_cast<T *>(v_to) + to);
}

// ---- pages_append ------------------------------------------------------------------------

// Rows of sequence b that can be appended, of its first `most`: those before the first
// whose place has no page. For all threads of the block.
__device__ inline uint32_t count_rows(const PagesAppendArgs &a, uint32_t b, uint32_t start, uint32_t most) {
    __shared__ uint32_t least;
    most = min(most, a.table * a.page - start);
    if (!most) return 0;
    if (threadIdx.x == 0) least = a.table;
    __syncthreads();
    const float *table = a.tables + size_t(b) * a.table;
    const uint32_t last = (start + most - 1) / a.page;
    uint32_t bad = a.table;
    for (uint32_t e = start / a.page + threadIdx.x; e <= last; e += kThreads)
        if (!is_whole(table[e], a.pages)) bad = min(bad, e);
    if (bad < a.table) atomicMin(&least, bad);
    __syncthreads();
    const uint32_t got = least;
    __syncthreads();
    return got > last ? most : got * a.page > start ? got * a.page - start : 0u;
}

__device__ inline uint32_t start_of(const PagesAppendArgs &a, uint32_t b) {
    return whole_below(a.lengths[b], a.table * a.page);
}

// Many rows: every sequence's new length by a launch of its own, so that the moving
// blocks need not look at all the pages before theirs.
__global__ __launch_bounds__(kThreads) void pages_count(PagesAppendArgs a) {
    const uint32_t b = blockIdx.x, start = start_of(a, b);
    const uint32_t count = count_rows(a, b, start, whole_below(a.counts[b], a.rows));
    if (threadIdx.x == 0) a.new_lengths[b] = float(start + count);
}

// A block takes `span` rows of a sequence, of all heads where rows come by token (`heads`
// is 1 then and `wide` all of a row), else of one head.
template <typename T, bool COUNTED>
__global__ __launch_bounds__(kThreads) void pages_append(PagesAppendArgs a, uint32_t heads, uint32_t wide, uint32_t span,
                                                         uint32_t spans, uint32_t items) {
    const uint32_t dim = a.dim * sizeof(float) / sizeof(T), row = a.kv_heads * dim;
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t at = item % spans, rest = item / spans, h = rest % heads, b = rest / heads;
        const uint32_t first = at * span, start = start_of(a, b);
        uint32_t count;
        if (COUNTED) {
            count = uint32_t(a.new_lengths[b]) - start;
        } else {
            // The first block of a sequence also writes its new length.
            const bool whole = h == 0 && at == 0;
            const uint32_t asked = whole_below(a.counts[b], a.rows);
            count = count_rows(a, b, start, whole ? asked : min(asked, first + span));
            if (whole && threadIdx.x == 0) a.new_lengths[b] = float(start + count);
        }
        if (count <= first) continue;
        const uint32_t n = min(count - first, span) * wide;
        const size_t from = (size_t(rest) * a.rows + first) * wide;
        const float *table = a.tables + size_t(b) * a.table;
#pragma unroll 2
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t r = i / wide, e = i - r * wide, t = start + first + r;
            const uint32_t entry = t / a.page, in = t - entry * a.page;
            const size_t page = uint32_t(table[entry]);
            size_t to;
            if (a.pages_token_major) {
                to = (page * a.page + in) * row + (a.token_major ? e : h * dim + e);
            } else {
                const uint32_t head = a.token_major ? e / dim : h;
                to = ((page * a.kv_heads + head) * a.page + in) * dim + (a.token_major ? e - head * dim : e);
            }
            move<T>(a.k, a.v, from + i, a.k_pages, a.v_pages, to);
        }
    }
}

// A block of the one-launch form looks at the entries of all the rows before its own. One
// sequence, 8 heads of 128, pages of 16, that form and the counted one: 131072 rows 444 and 418 us,
// 65536 203 and 206, 8192 27 and 30; 8 sequences of 131072 rows of 64 floats 229 and 217, of 32768
// 54.8 and 56.6.
constexpr uint32_t kCountedEntries = 4096;

struct Split {
    uint32_t heads, wide, span, spans;
    uint64_t items;
};
Split split_of(uint32_t batch, uint32_t kv_heads, uint32_t rows, uint32_t dim, bool token_major, bool vec) {
    Split s;
    s.heads = token_major ? 1 : kv_heads;
    s.wide = (token_major ? kv_heads * dim : dim) / (vec ? 4 : 1);
    s.span = s.wide < kBlockWords ? kBlockWords / s.wide : 1;
    s.spans = (rows + s.span - 1) / s.span;
    s.items = uint64_t(batch) * s.heads * s.spans;
    return s;
}

template <typename T>
hipError_t launch_append(hipStream_t stream, const PagesAppendArgs &a) {
    const Split s = split_of(a.batch, a.kv_heads, a.rows, a.dim, a.token_major, sizeof(T) == 16);
    const uint32_t items = uint32_t(s.items);
    const dim3 grid(items < kMaxBlocks ? items : kMaxBlocks), block(kThreads);
    if (a.rows / a.page > kCountedEntries) {
        hipLaunchKernelGGL(pages_count, dim3(a.batch), block, 0, stream, a);
        hipLaunchKernelGGL((pages_append<T, true>), grid, block, 0, stream, a, s.heads, s.wide, s.span, s.spans, items);
    } else {
        hipLaunchKernelGGL((pages_append<T, false>), grid, block, 0, stream, a, s.heads, s.wide, s.span, s.spans, items);
    }
    return hipGetLastError();
}

// ---- pages_copy --------------------------------------------------------------------------

// Float4s, or floats, of each tensor that a thread has on their way at once.
constexpr uint32_t kCopyWords = 4;

// `blocks` blocks for each copy. One whose target another reads, or an earlier one writes,
// is not made, so that the order in which blocks run changes nothing.
template <typename T>
__global__ __launch_bounds__(kThreads) void pages_copy(PagesCopyArgs a, uint32_t blocks) {
    const uint32_t c = blockIdx.x / blocks, part = blockIdx.x - c * blocks;
    const float source = a.sources[c], target = a.targets[c];
    if (!is_whole(source, a.pages) || !is_whole(target, a.pages) || !(a.copy_rows[c] >= 1.f)) return;
    const uint32_t rows = whole_below(a.copy_rows[c], a.page), dim = a.dim * sizeof(float) / sizeof(T);
    // Runs of rows that lie together: all heads of a token, or one head's tokens.
    const uint32_t runs = a.pages_token_major ? 1 : a.kv_heads, run = rows * dim * (a.pages_token_major ? a.kv_heads : 1);
    const size_t page = size_t(a.page) * a.kv_heads * dim, pitch = size_t(a.page) * dim;
    const uint32_t pieces = (run + kCopyWords * kThreads - 1) / (kCopyWords * kThreads);
    if (part >= runs * pieces) return;
    for (uint32_t i = part; i < runs * pieces; i += blocks) {
        const uint32_t h = i / pieces, at = (i - h * pieces) * kCopyWords * kThreads + threadIdx.x;
        const size_t from = size_t(source) * page + h * pitch + at, to = size_t(target) * page + h * pitch + at;
        T k[kCopyWords], v[kCopyWords];
#pragma unroll
        for (uint32_t x = 0; x < kCopyWords; ++x)
            if (at + x * kThreads < run) {
                k[x] = __builtin_nontemporal_load(reinterpret_cast<const T *>(a.k_pages) + from + x * kThreads);
                v[x] = __builtin_nontemporal_load(reinterpret_cast<const T *>(a.v_pages) + from + x * kThreads);
            }
        if (i == part) {  // asked while the first rows are on their way
            bool clash = false;
#pragma unroll 4
            for (uint32_t j = threadIdx.x; j < a.copies; j += kThreads) {
                const float from = a.sources[j], to = a.targets[j], n = a.copy_rows[j];
                clash |= ((from == target) | ((j < c) & (to == target))) & is_whole(from, a.pages) & is_whole(to, a.pages) & (n >= 1.f);
            }
            if (__syncthreads_or(clash)) return;
        }
#pragma unroll
        for (uint32_t x = 0; x < kCopyWords; ++x)
            if (at + x * kThreads < run) {
                __builtin_nontemporal_store(k[x], reinterpret_cast<T *>(a.k_pages) + to + x * kThreads);
                __builtin_nontemporal_store(v[x], reinterpret_cast<T *>(a.v_pages) + to + x * kThreads);
            }
    }
}

// Blocks of a copy: as many as there is work for, but no more than fill the chip.
constexpr uint32_t kCopyBlocks = 16384;
uint32_t copy_blocks(uint32_t copies, uint32_t page, uint32_t kv_heads, uint32_t dim) {
    const uint64_t words = uint64_t(page) * kv_heads * dim / (dim % 4 ? 1 : 4);
    const uint64_t piece = kCopyWords * kThreads, share = (kCopyBlocks + copies - 1) / copies;
    const uint64_t most = (words + piece - 1) / piece;
    return uint32_t(most < share ? most : share);
}

// ---- pages_fork --------------------------------------------------------------------------

constexpr uint32_t kForkPages = 4 * kThreads;  // pages of a block

// The workspace, in 32-bit words.
struct ForkSpace {
    int *sums;                                // what each page's uses gain; zeros between calls
    uint32_t *keep, *need, *before, *counts;  // of a sequence; needs before it (and in all); free pages of a block
};
__host__ __device__ inline uint32_t fork_blocks(uint32_t pages) { return (pages + kForkPages - 1) / kForkPages; }
__host__ __device__ inline ForkSpace fork_space(float *workspace, uint32_t pages, uint32_t batch) {
    uint32_t *const w = reinterpret_cast<uint32_t *>(workspace), *const per = w + pages;
    return {reinterpret_cast<int *>(w), per, per + batch, per + 2 * size_t(batch), per + 3 * size_t(batch) + 1};
}

// A whole number of 0 .. batch - 1, or batch.
__device__ inline uint32_t parent_of(const PagesForkArgs &a, uint32_t s) {
    return is_whole(a.parents[s], a.batch) ? uint32_t(a.parents[s]) : a.batch;
}

// A table's entries that a thread keeps in registers (of kThreads at a time); -1 past the
// table, or where it names no page. Those of longer tables are read again where they are used:
// 512 sequences with tables of 1024, 2048, 2304 and 4096 entries 23.7, 29.5, 31.7 and 44.9 us.
constexpr uint32_t kNearEntries = 8;
struct Entries {
    float x[kNearEntries];
};
__device__ inline Entries near_entries(const PagesForkArgs &a, const float *table) {
    Entries e;
#pragma unroll
    for (uint32_t i = 0; i < kNearEntries; ++i) {
        const uint32_t at = threadIdx.x + i * kThreads;
        e.x[i] = at < a.table ? table[at] : -1.f;
    }
    return e;
}
// The first of this thread's entries that names no page, or the table's end.
__device__ inline uint32_t first_gap(const PagesForkArgs &a, const float *table, const Entries &e) {
    uint32_t bad = a.table;
    for (uint32_t at = threadIdx.x + kNearEntries * kThreads; at < a.table; at += kThreads)
        if (!is_whole(table[at], a.pages)) bad = min(bad, at);
#pragma unroll
    for (uint32_t i = 0; i < kNearEntries; ++i)
        if (!is_whole(e.x[i], a.pages)) bad = min(bad, threadIdx.x + i * kThreads);
    return bad;
}

__global__ __launch_bounds__(kThreads) void pages_fork_tables(PagesForkArgs a) {
    __shared__ uint32_t children, older, held, theirs;
    const ForkSpace w = fork_space(a.workspace, a.pages, a.batch);
    const uint32_t s = blockIdx.x, parent = parent_of(a, s), tid = threadIdx.x;
    const bool alive = parent < a.batch;
    const float *const table = a.tables + size_t(s) * a.table;
    const float *const from = a.tables + size_t(alive ? parent : s) * a.table;
    // Everything that is read, at once: both tables and who goes on from whom.
    const Entries mine = near_entries(a, table), yours = near_entries(a, from);
    const float my_length = a.lengths[s], your_length = a.lengths[alive ? parent : s], reserve = a.reserve[s];
    uint32_t going = 0, before = 0;
    for (uint32_t i = tid; i < a.batch; i += kThreads) {
        const uint32_t p = parent_of(a, i);
        going += p == s;
        before += p == parent && i < s;
    }
    if (tid == 0) {
        children = older = 0;
        held = theirs = a.table;
    }
    __syncthreads();
    // Pages of a table: those before its first entry that names none.
    const uint32_t gap = first_gap(a, table, mine), your_gap = first_gap(a, from, yours);
    if (gap < a.table) atomicMin(&held, gap);
    if (your_gap < a.table) atomicMin(&theirs, your_gap);
    if (going) atomicAdd(&children, going);
    if (before) atomicAdd(&older, before);
    __syncthreads();
    {
        // This sequence's pages: whole ones for each child, the others for its first.
        const uint32_t length = min(whole_below(my_length, a.table * a.page), held * a.page), full = length / a.page;
        const int n = int(children);
        auto gain = [&](uint32_t e, float page) {
            const int more = (e < full ? n : min(n, 1)) - 1;
            if (e < held && more) atomicAdd(w.sums + uint32_t(page), more);
        };
        if (n != 1) {
#pragma unroll
            for (uint32_t i = 0; i < kNearEntries; ++i) gain(tid + i * kThreads, mine.x[i]);
            for (uint32_t e = tid + kNearEntries * kThreads; e < held; e += kThreads) gain(e, table[e]);
        }
    }
    float *const to = a.new_tables + size_t(s) * a.table;
    uint32_t keep = 0, need = 0, length = 0, part = 0, full = 0;
    if (alive) {
        length = min(whole_below(your_length, a.table * a.page), theirs * a.page);
        full = length / a.page;
        keep = older ? full : theirs;
        if (older) part = length - full * a.page;
        const uint64_t end = uint64_t(length) + whole_below(reserve, a.table * a.page);
        const uint32_t want = uint32_t(min(uint64_t(a.table), (end + a.page - 1) / a.page));
        need = want > keep ? want - keep : 0;
    }
    auto inherit = [&](uint32_t e, float page) {
        to[e] = e < keep ? page : -1.f;
        if (part && e == full) a.sources[s] = page;  // its partial page, which this sequence gets a copy of
    };
#pragma unroll
    for (uint32_t i = 0; i < kNearEntries; ++i)
        if (tid + i * kThreads < a.table) inherit(tid + i * kThreads, yours.x[i]);
    for (uint32_t e = tid + kNearEntries * kThreads; e < a.table; e += kThreads) inherit(e, from[e]);
    if (tid == 0) {
        w.keep[s] = keep;
        w.need[s] = need;
        a.new_lengths[s] = float(length);
        a.copy_rows[s] = float(part);
        if (!part) a.sources[s] = -1.f;
    }
}

// Sum over the block's threads up to and with this one; `total` of all.
__device__ inline uint32_t block_scan(uint32_t x, uint32_t &total) {
    __shared__ uint32_t waves[kThreads / 64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    if (lane == 63) waves[wave] = x;
    __syncthreads();
    total = 0;
#pragma unroll
    for (uint32_t i = 0; i < kThreads / 64; ++i) {
        if (i < wave) x += waves[i];
        total += waves[i];
    }
    __syncthreads();
    return x;
}

__global__ __launch_bounds__(kThreads) void pages_fork_count(PagesForkArgs a) {
    const ForkSpace w = fork_space(a.workspace, a.pages, a.batch);
    const uint32_t blocks = fork_blocks(a.pages);
    uint32_t total;
    if (blockIdx.x < blocks) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t p = blockIdx.x * kForkPages + i * kThreads + threadIdx.x;
            if (p >= a.pages) break;
            const int more = w.sums[p];
            const float uses = a.uses[p] + float(more);
            a.new_uses[p] = uses;
            if (more) w.sums[p] = 0;
            n += uses == 0.f;
        }
        block_scan(n, total);
        if (threadIdx.x == 0) w.counts[blockIdx.x] = total;
        return;
    }
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < a.batch; s0 += kThreads) {
        const uint32_t s = s0 + threadIdx.x, mine = s < a.batch ? w.need[s] : 0u;
        const uint32_t up_to = block_scan(mine, total);
        // A pool has at most 2^24 pages; sums that pass it need not be told apart.
        if (s < a.batch) w.before[s] = before + up_to - mine;
        before = min(before + total, 1u << 30);
    }
    if (threadIdx.x == 0) w.before[a.batch] = before;
}

constexpr uint32_t kNearNeeds = 2048;

__global__ __launch_bounds__(kThreads) void pages_fork_allot(PagesForkArgs a) {
    __shared__ uint32_t needs[kNearNeeds];
    const ForkSpace w = fork_space(a.workspace, a.pages, a.batch);
    const uint32_t blocks = fork_blocks(a.pages), asked = w.before[a.batch];
    const bool pages = blockIdx.x < blocks;
    // Everything that is read, at once: four neighbouring pages a thread, the free ones of the
    // blocks before (of a block of sequences: of all), and for the search below the sums of
    // needs, in LDS where they fit.
    const uint32_t first = blockIdx.x * kForkPages + 4 * threadIdx.x;
    const bool fits = a.batch <= kNearNeeds;
    bool open[4];
    uint32_t free = 0, before = 0, n = 0;
    if (pages) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            open[i] = first + i < a.pages && a.new_uses[first + i] == 0.f;
            n += open[i];
        }
        if (fits)
            for (uint32_t s = threadIdx.x; s < a.batch; s += kThreads) needs[s] = w.before[s];
    }
    for (uint32_t i = threadIdx.x; i < (pages ? blockIdx.x : blocks); i += kThreads) before += w.counts[i];
    block_scan(before, free);
    if (!pages) {
        const uint32_t s = (blockIdx.x - blocks) * kThreads + threadIdx.x;
        if (s >= a.batch) return;
        const uint32_t start = w.before[s], need = w.need[s], got = start < free ? min(need, free - start) : 0u;
        a.missing[s] = float(need - got);
        const bool copy = a.copy_rows[s] > 0.f;
        if (!copy || !got) a.targets[s] = -1.f;
        if (copy && !got) {  // without the page that its partial one would go to
            a.new_lengths[s] = float(w.keep[s] * a.page);
            a.copy_rows[s] = 0.f;
            a.sources[s] = -1.f;
        }
        return;
    }
    if (free >= asked) return;
    uint32_t total, rank = free + block_scan(n, total) - n;
    for (uint32_t i = 0; i < 4; ++i) {
        if (!open[i]) continue;
        if (rank >= asked) return;
        // The last sequence with `before` at most rank has a need past it.
        uint32_t lo = 0, hi = a.batch - 1;
        while (lo < hi) {
            const uint32_t mid = (lo + hi + 1) / 2;
            if ((fits ? needs[mid] : w.before[mid]) <= rank)
                lo = mid;
            else
                hi = mid - 1;
        }
        const uint32_t place = w.keep[lo] + rank - w.before[lo];
        a.new_tables[size_t(lo) * a.table + place] = float(first + i);
        a.new_uses[first + i] = 1.f;
        if (rank == w.before[lo] && a.copy_rows[lo] > 0.f) a.targets[lo] = float(first + i);
        ++rank;
    }
}

// Few sequences over few pages: the same by one block, with tables and sums in LDS. 4
// sequences with tables of 64 entries and 232 pages: 11.3 us by three launches, 5.1 so; 64
// such sequences and 8000 pages 15.6 and 12.6.
constexpr uint32_t kSmallBatch = 64, kSmallEntries = 4096, kSmallPages = 8192, kSmallThreads = 1024;
inline bool is_small(uint32_t batch, uint32_t pages, uint32_t table) {
    return batch <= kSmallBatch && uint64_t(batch) * table <= kSmallEntries && pages <= kSmallPages;
}

__global__ __launch_bounds__(kSmallThreads) void pages_fork_small(PagesForkArgs a) {
    constexpr uint32_t kEntries = kSmallEntries / kSmallThreads, kPages = kSmallPages / kSmallThreads;
    __shared__ float old_tables[kSmallEntries], new_tables[kSmallEntries];
    __shared__ int sums[kSmallPages];
    __shared__ uint32_t parents[kSmallBatch], children[kSmallBatch], eldest[kSmallBatch], held[kSmallBatch], lengths[kSmallBatch];
    __shared__ uint32_t keep[kSmallBatch], needs[kSmallBatch], before[kSmallBatch + 1], waves[kSmallThreads / 64];
    __shared__ uint32_t full[kSmallBatch], parts[kSmallBatch], targets[kSmallBatch];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid / 64, entries = a.batch * a.table;
    // Everything that is read, at once.
    float near[kEntries], uses[kPages];
#pragma unroll
    for (uint32_t i = 0; i < kEntries; ++i) {
        const uint32_t e = tid + i * kSmallThreads;
        near[i] = e < entries ? a.tables[e] : -1.f;
    }
    // A thread has neighbouring pages, so that free ones are counted in order.
    const uint32_t first = tid * kPages;
    const bool whole = first + kPages <= a.pages;
    if (whole) {
#pragma unroll
        for (uint32_t i = 0; i < kPages; i += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(a.uses + first + i);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) uses[i + e] = x[e];
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kPages; ++i) uses[i] = first + i < a.pages ? a.uses[first + i] : 1.f;
    }
    float reserve = 0.f;
    if (tid < a.batch) {
        reserve = a.reserve[tid];
        parents[tid] = parent_of(a, tid);
        lengths[tid] = whole_below(a.lengths[tid], a.table * a.page);
        children[tid] = 0;
        eldest[tid] = a.batch;
        held[tid] = a.table;
        targets[tid] = a.pages;
    }
    for (uint32_t i = tid; i < a.pages; i += kSmallThreads) sums[i] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kEntries; ++i) {
        const uint32_t e = tid + i * kSmallThreads, s = e / a.table;
        if (e >= entries) break;
        old_tables[e] = near[i];
        if (!is_whole(near[i], a.pages)) atomicMin(&held[s], e - s * a.table);
    }
    if (tid < a.batch && parents[tid] < a.batch) {
        atomicAdd(&children[parents[tid]], 1u);
        atomicMin(&eldest[parents[tid]], tid);
    }
    __syncthreads();
    if (tid < a.batch) {
        lengths[tid] = min(lengths[tid], held[tid] * a.page);
        full[tid] = lengths[tid] / a.page;
    }
    __syncthreads();
    if (wave == 0) {
        uint32_t need = 0;
        if (tid < a.batch) {
            const uint32_t p = parents[tid];
            uint32_t kept = 0, part = 0;
            if (p < a.batch) {
                const bool first = eldest[p] == tid;
                kept = first ? held[p] : full[p];
                if (!first) part = lengths[p] - full[p] * a.page;
                const uint64_t end = uint64_t(lengths[p]) + whole_below(reserve, a.table * a.page);
                const uint32_t want = uint32_t(min(uint64_t(a.table), (end + a.page - 1) / a.page));
                need = want > kept ? want - kept : 0;
            }
            keep[tid] = kept;
            parts[tid] = part;
            needs[tid] = need;
        }
        uint32_t sum = need;
#pragma unroll
        for (uint32_t d = 1; d < 64; d *= 2) {
            const uint32_t y = __shfl_up(sum, d);
            if (lane >= d) sum += y;
        }
        if (tid < a.batch) before[tid] = sum - need;
        if (lane == 63) before[a.batch] = sum;
    }
    // What each page's uses gain.
#pragma unroll
    for (uint32_t i = 0; i < kEntries; ++i) {
        const uint32_t e = tid + i * kSmallThreads, s = e / a.table, at = e - s * a.table;
        if (e >= entries) break;
        const int n = int(children[s]), more = (at < full[s] ? n : min(n, 1)) - 1;
        if (at < held[s] && more) atomicAdd(&sums[uint32_t(near[i])], more);
    }
    __syncthreads();
    const uint32_t asked = before[a.batch];
#pragma unroll
    for (uint32_t i = 0; i < kEntries; ++i) {
        const uint32_t e = tid + i * kSmallThreads, s = e / a.table, at = e - s * a.table;
        if (e >= entries) break;
        new_tables[e] = at < keep[s] ? old_tables[parents[s] * a.table + at] : -1.f;
    }
    uint32_t n = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPages; ++i) {
        if (first + i < a.pages) uses[i] += float(sums[first + i]);
        n += first + i < a.pages && uses[i] == 0.f;
    }
    uint32_t rank = n;
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_up(rank, d);
        if (lane >= d) rank += y;
    }
    if (lane == 63) waves[wave] = rank;
    __syncthreads();
    uint32_t free = 0;
#pragma unroll
    for (uint32_t i = 0; i < kSmallThreads / 64; ++i) {
        if (i < wave) rank += waves[i];
        free += waves[i];
    }
    rank -= n;
#pragma unroll
    for (uint32_t i = 0; i < kPages; ++i) {
        if (first + i >= a.pages || uses[i] != 0.f) continue;
        if (rank < asked) {
            // The last sequence with `before` at most rank has a need past it.
            uint32_t lo = 0, hi = a.batch - 1;
            while (lo < hi) {
                const uint32_t mid = (lo + hi + 1) / 2;
                if (before[mid] <= rank)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            new_tables[lo * a.table + keep[lo] + rank - before[lo]] = float(first + i);
            if (rank == before[lo]) targets[lo] = first + i;
            uses[i] = 1.f;
        }
        ++rank;
    }
    if (whole) {
#pragma unroll
        for (uint32_t i = 0; i < kPages; i += 4)
            *reinterpret_cast<f32x4 *>(a.new_uses + first + i) = f32x4{uses[i], uses[i + 1], uses[i + 2], uses[i + 3]};
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kPages; ++i)
            if (first + i < a.pages) a.new_uses[first + i] = uses[i];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kEntries; ++i) {
        const uint32_t e = tid + i * kSmallThreads;
        if (e < entries) a.new_tables[e] = new_tables[e];
    }
    if (tid < a.batch) {
        const uint32_t p = parents[tid], start = before[tid], need = needs[tid], got = start < free ? min(need, free - start) : 0u;
        const bool copy = parts[tid] && got;
        a.missing[tid] = float(need - got);
        a.new_lengths[tid] = p == a.batch ? 0.f : float(parts[tid] && !got ? full[p] * a.page : lengths[p]);
        a.sources[tid] = copy ? old_tables[p * a.table + full[p]] : -1.f;
        a.targets[tid] = copy ? float(targets[tid]) : -1.f;
        a.copy_rows[tid] = copy ? float(parts[tid]) : 0.f;
    }
}

}  // namespace

LaunchShape pages_append_shape(uint32_t batch, uint32_t kv_heads, uint32_t rows, uint32_t page, uint32_t dim,
                               bool token_major) {
    const uint64_t items = split_of(batch, kv_heads, rows, dim, token_major, dim % 4 == 0).items;
    if (items > 0xfffffffeull - kMaxBlocks) return {nullptr, {0, 0, 0}, {0, 0, 0}, 0};
    return {rows / page > kCountedEntries ? "pages_append_counted" : "pages_append",
            {uint32_t(items < kMaxBlocks ? items : kMaxBlocks), 1, 1}, {kThreads, 1, 1}, uint32_t(sizeof(uint32_t))};
}

hipError_t pages_append_f32(hipStream_t stream, const PagesAppendArgs &a) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                           reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages);
    if (a.dim % 4 == 0 && bits & 15u) return hipErrorInvalidValue;  // the runtime's regions are aligned
    return a.dim % 4 == 0 ? launch_append<f32x4>(stream, a) : launch_append<float>(stream, a);
}

LaunchShape pages_copy_shape(uint32_t copies, uint32_t kv_heads, uint32_t page, uint32_t dim) {
    const uint64_t blocks = uint64_t(copies) * copy_blocks(copies, page, kv_heads, dim);
    // A page is counted in 32 bits.
    if (uint64_t(page) * kv_heads * dim > 0x7fffffffull) return {nullptr, {0, 0, 0}, {0, 0, 0}, 0};
    return {"pages_copy", {uint32_t(blocks), 1, 1}, {kThreads, 1, 1}, 0};
}

hipError_t pages_copy_f32(hipStream_t stream, const PagesCopyArgs &a) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages);
    if (a.dim % 4 == 0 && bits & 15u) return hipErrorInvalidValue;
    const uint32_t blocks = copy_blocks(a.copies, a.page, a.kv_heads, a.dim);
    const dim3 grid(a.copies * blocks);
    if (a.dim % 4 == 0)
        hipLaunchKernelGGL(pages_copy<f32x4>, grid, dim3(kThreads), 0, stream, a, blocks);
    else
        hipLaunchKernelGGL(pages_copy<float>, grid, dim3(kThreads), 0, stream, a, blocks);
    return hipGetLastError();
}

LaunchShape pages_fork_shape(uint32_t batch, uint32_t pages, uint32_t table) {
    if (is_small(batch, pages, table))
        return {"pages_fork_small", {1, 1, 1}, {kSmallThreads, 1, 1},
                uint32_t(sizeof(float) * (2 * kSmallEntries + kSmallPages + 11 * kSmallBatch + 1 + kSmallThreads / 64))};
    return {"pages_fork", {batch, 1, 1}, {kThreads, 1, 1}, uint32_t(4 * sizeof(uint32_t))};
}

size_t pages_fork_workspace_bytes(uint32_t batch, uint32_t pages, uint32_t table) {
    if (is_small(batch, pages, table)) return 0;
    return (size_t(pages) + 3 * size_t(batch) + 1 + fork_blocks(pages)) * sizeof(uint32_t);
}

hipError_t pages_fork_f32(hipStream_t stream, const PagesForkArgs &a) {
    if (is_small(a.batch, a.pages, a.table)) {
        if ((reinterpret_cast<uintptr_t>(a.uses) | reinterpret_cast<uintptr_t>(a.new_uses)) & 15u) return hipErrorInvalidValue;
        hipLaunchKernelGGL(pages_fork_small, dim3(1), dim3(kSmallThreads), 0, stream, a);
        return hipGetLastError();
    }
    if (!a.workspace) return hipErrorInvalidValue;
    const uint32_t blocks = fork_blocks(a.pages);
    hipLaunchKernelGGL(pages_fork_tables, dim3(a.batch), dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL(pages_fork_count, dim3(blocks + 1), dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL(pages_fork_allot, dim3(blocks + (a.batch + kThreads - 1) / kThreads), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace hipk
}  // namespace jade
