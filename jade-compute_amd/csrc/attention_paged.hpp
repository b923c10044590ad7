// Attention over a paged cache: arguments, and the device parts that its kernels share:
// where a run's tiles lie, and how a row's sums become outputs or go to the workspace.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "whole.hpp"

namespace jade {
namespace hipk {

// Strides in elements. Rows of q and out are [batch, head, query]; a page's row of a head
// is at page * p_page + kv head * p_head + row * p_row.
struct PagedArgs {
    const float *q, *k, *v, *tables, *lengths, *counts;
    float *out, *partial;
    size_t q_batch, q_head, p_page, p_head;
    uint32_t q_row, p_row;
    uint32_t batch, kv_heads, group, queries, pages, table, page, dim;
    uint32_t steps, inverse;  // 16-token steps of a page; 2^31 / steps, rounded up
    uint32_t least_rows, most_rows;  // of a kv head, of the sequences that a launch takes
    uint32_t runs;
    bool uncut;    // no run ends inside a (sequence, kv head, row block)
    float qscale;  // scale * log2(e)
};

// The kernel on bf16 parts (attention_paged_flash.hip). Needs dim % 4 == 0 and at most 128,
// 16-byte aligned tensors and a sequence's rows of q below 2 GiB.
constexpr uint32_t kPagedFlashTile = 32;
inline uint32_t paged_flash_rows(uint32_t dim) { return dim <= 64 ? 128 : 256; }
void launch_paged_flash(hipStream_t stream, const PagedArgs &args);
uint32_t paged_flash_lds_bytes(uint32_t dim);

namespace {
namespace paged {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;
constexpr uint32_t kCus = 256;
constexpr float kLazyMax = 8.0f;   // log2 units: the running maximum moves only past this
constexpr uint32_t kRawBuffer = 0x00020000;    // buffer descriptor word 3: raw buffer, 32-bit data format
constexpr uint32_t kDeadOffset = 0x80000000u;  // past every descriptor's end: reads zero
constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kNoPage = ~0u;

__device__ inline uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline uint32_t of_lane(uint32_t x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

// Sum over the lanes up to and with this one: within the rows of 16 by shifts, then
// each row's last lane into the rows after it.
__device__ inline uint32_t scan_add(uint32_t x) {
#define JADE_SCAN(control, rows) x += __builtin_amdgcn_update_dpp(0, x, control, rows, 0xf, false)
    JADE_SCAN(0x111, 0xf);
    JADE_SCAN(0x112, 0xf);
    JADE_SCAN(0x114, 0xf);
    JADE_SCAN(0x118, 0xf);
    JADE_SCAN(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
    JADE_SCAN(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef JADE_SCAN
    return x;
}

__device__ inline float across_keys_max(float x) {
    return fmaxf(fmaxf(x, __shfl_xor(x, 16)), fmaxf(__shfl_xor(x, 32), __shfl_xor(x, 48)));
}
__device__ inline float across_keys_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// Run of block `id`: the runs of one XCD are neighbours.
__device__ inline uint32_t run_of(uint32_t id, uint32_t runs) { return id % 8 * (runs / 8) + id / 8; }

// A sequence: its tokens, the new ones among them, and what they make of blocks of rows (for
// each kv head) and tiles of keys (for each block, as many as its last query sees). Row r of
// a kv head is head r % group of the group and query r / group, so that a block of rows has
// neighbouring queries, and sequences of few new tokens have few blocks.
struct Sequence {
    uint32_t length, count;
};
// A (kv head, row block) of a sequence, a place among its tiles and how many those are.
struct Spot {
    uint32_t kv, rb, tile, tiles;
};
template <int TILE, int RB>
struct Work {
    const PagedArgs &a;
    const Sequence near;         // sequence (lane)
    const uint32_t own, up_to;   // its tiles, of all kv heads and row blocks; those up to it
    uint32_t total;

    __device__ Sequence load(uint32_t b) const {
        const uint32_t i = min(b, a.batch - 1);  // no branch, so that loads of several are on their way at once
        const uint32_t length = whole_below(a.lengths[i], a.table * a.page), count = whole_below(a.counts[i], a.queries);
        return b < a.batch ? Sequence{length, count} : Sequence{0, 0};
    }
    // Whether there is anything to do, by this launch.
    __device__ bool active(const Sequence &s) const {
        const uint32_t rows = s.count * a.group;
        return s.length && rows >= a.least_rows && rows <= a.most_rows;
    }
    __device__ uint32_t blocks(const Sequence &s) const { return active(s) ? (s.count * a.group + RB - 1) / RB : 0u; }
    // Tiles that row block rb sees any key of; one where there is none, for the rows' zeros.
    __device__ uint32_t tiles(const Sequence &s, uint32_t rb) const {
        const int seen = int(s.length) - int(s.count) + int(min(s.count, (rb * RB + RB - 1) / a.group + 1));
        return seen > TILE ? uint32_t(seen + TILE - 1) / TILE : 1u;
    }
    __device__ uint32_t tiles_a_head(const Sequence &s) const {
        const uint32_t n = blocks(s);
        if (n <= 1) return n ? (s.length + TILE - 1) / TILE : 0u;
        uint32_t sum = 0;
        for (uint32_t rb = 0; rb < n; ++rb) sum += tiles(s, rb);
        return sum;
    }
    __device__ uint32_t all_of(const Sequence &s) const { return tiles_a_head(s) * a.kv_heads; }
    // Place `in` of a sequence's tiles, `all` of them.
    __device__ Spot spot(const Sequence &s, uint32_t all, uint32_t in) const {
        const uint32_t head = all / a.kv_heads, n = blocks(s);
        Spot p;
        p.kv = in / head;
        p.rb = 0;
        p.tile = in - p.kv * head;
        p.tiles = head;
        if (n > 1)
            for (;; p.rb += 64) {
                const uint32_t rb = p.rb + (threadIdx.x & 63), mine = rb < n ? tiles(s, rb) : 0u, sum = scan_add(mine);
                const uint64_t past = __ballot(sum > p.tile);
                if (past) {
                    const int first = __builtin_ctzll(past);
                    p.rb += first;
                    p.tile -= of_lane(sum - mine, first);
                    p.tiles = of_lane(mine, first);
                    break;
                }
                p.tile -= of_lane(sum, 63);
            }
        return p;
    }
    // The tiles of one kv head before row block rb.
    __device__ uint32_t tiles_before(const Sequence &s, uint32_t rb) const {
        uint32_t sum = 0;
        for (uint32_t first = 0; first < rb; first += 64) {
            const uint32_t x = first + (threadIdx.x & 63);
            sum += of_lane(scan_add(x < rb ? tiles(s, x) : 0u), 63);
        }
        return sum;
    }
    // All tiles of sequence b, s.
    __device__ uint32_t all_at(uint32_t b, const Sequence &s) const {
        return b < 64 ? of_lane(own, int(b)) : uniform(all_of(s));
    }
    // Of one sequence, for the whole wave.
    __device__ Sequence at(uint32_t b) const {
        return b < 64 ? Sequence{of_lane(near.length, int(b)), of_lane(near.count, int(b))} : anew(b);
    }
    // The same from memory: no register keeps the near ones for it.
    __device__ Sequence anew(uint32_t b) const {
        const Sequence s = load(b);
        return {uniform(s.length), uniform(s.count)};
    }
    __device__ explicit Work(const PagedArgs &args)
        : a(args), near(load(threadIdx.x & 63)), own(all_of(near)), up_to(scan_add(own)), total(of_lane(up_to, 63)) {
        for (uint32_t b0 = 64; b0 < a.batch; b0 += 64) total += of_lane(scan_add(lane_work(b0)), 63);
    }
    // This lane's work among the sequences from b0 on.
    __device__ uint32_t lane_work(uint32_t b0) const { return all_of(load(b0 + (threadIdx.x & 63))); }
    // The sequence that tile t < total belongs to, and the tiles before it.
    __device__ void find(uint32_t t, uint32_t &b, uint32_t &before) const {
        before = 0;
        uint32_t sum = up_to, mine = own;
        Sequence next{0, 0};
        if (a.batch > 64) next = load(64 + (threadIdx.x & 63));
        for (b = 0;; b += 64, mine = all_of(next), sum = scan_add(mine), next = load(b + 64 + (threadIdx.x & 63))) {
            const uint64_t past = __ballot(before + sum > t);
            if (past) {
                const int first = __builtin_ctzll(past);
                b += first;
                before += of_lane(sum - mine, first);
                return;
            }
            before += of_lane(sum, 63);
        }
    }
    // Where run `run` starts: tile run * chunk, but at the nearest end of a (kv head, row
    // block) where a run has four or more whole ones of that sequence, or none is to be cut:
    // then none of them needs joining. `b` and `before` as find() leaves them; at the last tile's end they say
    // nothing.
    __device__ uint32_t start(uint32_t run, uint32_t chunk, uint32_t &b, uint32_t &before) const {
        const uint64_t at = uint64_t(run) * chunk;
        if (at >= total) return total;
        uint32_t t = uint32_t(at);
        find(t, b, before);
        const Sequence s = this->at(b);
        if (!rounds(s, chunk)) return t;
        const uint32_t all = all_at(b, s);
        const Spot p = spot(s, all, t - before);
        t = 2 * p.tile < p.tiles ? t - p.tile : t - p.tile + p.tiles;
        if (t == before + all) {
            before += all;
            ++b;
        }
        return t;
    }
    // The (kv head, row block)s of all sequences: number n's sequence and its number there, and
    // the tiles before that sequence; false past the last.
    __device__ uint32_t units_of(const Sequence &s) const { return blocks(s) * a.kv_heads; }
    __device__ bool find_unit(uint32_t n, uint32_t &b, uint32_t &unit, uint32_t &before) const {
        before = 0;
        uint32_t mine = units_of(near), tiles_up_to = up_to, tiles_mine = own;
        for (b = 0; b < a.batch; b += 64) {
            if (b) {
                const Sequence s = load(b + (threadIdx.x & 63));
                mine = units_of(s);
                tiles_mine = all_of(s);
                tiles_up_to = scan_add(tiles_mine);
            }
            const uint32_t sum = scan_add(mine);
            const uint64_t past = __ballot(sum > n);
            if (past) {
                const int first = __builtin_ctzll(past);
                b += first;
                unit = n - of_lane(sum - mine, first);
                before += of_lane(tiles_up_to - tiles_mine, first);
                return true;
            }
            n -= of_lane(sum, 63);
            before += of_lane(tiles_up_to, 63);
        }
        return false;
    }
    // No run ends inside a row block of the sequence: where a run has four or more whole ones
    // (by the longest, so that all are cut alike); and on parts, whose cuts leave the sums of
    // 128 or 256 rows, where a block is short and no more than two runs (16 sequences of 64 to
    // 128 keys, 8 kv heads of 64, 400 rows each: 42.8 us cut, 26.6 whole).
    __device__ bool rounds(const Sequence &s, uint32_t chunk) const {
        const uint32_t n = (s.length + TILE - 1) / TILE;
        return a.uncut || 4 * n <= chunk || (TILE == int(kPagedFlashTile) && n <= 8 && n <= 2 * chunk);
    }
};

// Dims d .. d + 3 of a row, zeros from `dim` on and for no row. VEC: dim % 4 == 0 and
// 16-byte rows.
template <bool VEC>
__device__ inline f32x4 load_dims(const float *row, int d, int dim) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (VEC) {
        if (row && d < dim) x = *reinterpret_cast<const f32x4 *>(row + d);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (row && d + e < dim) x[e] = row[d + e];
    }
    return x;
}
template <bool VEC>
__device__ inline void store_dims(float *row, int d, int dim, f32x4 x) {
    if (VEC) {
        if (d < dim) *reinterpret_cast<f32x4 *>(row + d) = x;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < dim) row[d + e] = x[e];
    }
}

// The lane's number, made anew: what is computed from it is not kept in registers from
// outside a main loop.
__device__ inline int lane_now() {
    int l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(l));
    return l;
}

// The kernel's arguments where they were passed, read anew: nothing made of them is kept in
// registers across a main loop that has none to spare. Only in a kernel itself: a function
// that is called has no such place, and reads at 0.
typedef const __attribute__((address_space(4))) PagedArgs Args;
__device__ __attribute__((always_inline)) inline Args *args_now() {
    Args *p = reinterpret_cast<Args *>(reinterpret_cast<uintptr_t>(__builtin_amdgcn_kernarg_segment_ptr()));
    asm volatile("" : "+s"(p));
    return p;
}

// Row r of (sequence b, kv head), from its first dim, in q and out.
__device__ inline size_t row_at(const PagedArgs &a, uint32_t b, uint32_t kv, uint32_t r) {
    const uint32_t query = r / a.group, head = r - query * a.group;
    return size_t(b) * a.q_batch + (size_t(kv) * a.group + head) * a.q_head + size_t(query) * a.q_row;
}

// The 16 tokens from 16 n on of sequence b: their place in its table.
struct Place {
    uint32_t entry, step;  // of 16 tokens within the page
};
template <class Args>
__device__ inline Place place_of(const Args &a, uint32_t n) {
    const uint32_t entry = uint32_t(uint64_t(n) * a.inverse >> 31);
    return {entry, n - entry * a.steps};
}
template <class Args>
__device__ inline uint32_t page_of(const Args &a, float entry) {
    return entry >= 0.f && entry < float(a.pages) && entry == truncf(entry) ? uint32_t(entry) : kNoPage;
}

// Zeros for the rows that no launch has tiles for: those of queries past a sequence's count,
// and all of one without tokens. Row by row over the grid's waves.
template <int TILE, int RB>
__device__ inline void clear_rows(const Work<TILE, RB> &work) {
    const PagedArgs &a = work.a;
    const uint32_t lane = threadIdx.x & 63, wide = a.kv_heads * a.group * a.dim, waves = a.runs * kWaves;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
        const Sequence s = b0 ? work.load(b0 + lane) : work.near;
        const uint32_t kept = s.length ? s.count : 0u, rows = b0 + lane < a.batch ? a.queries - kept : 0u;
        const uint32_t sum = scan_add(rows), all = of_lane(sum, 63);
        for (uint32_t i = blockIdx.x * kWaves + uniform(threadIdx.x >> 6); i < all; i += waves) {
            const int at = __builtin_ctzll(__ballot(sum > i));
            const uint32_t query = of_lane(kept, at) + (i - of_lane(sum - rows, at));
            float *const out = a.out + size_t(b0 + at) * a.q_batch + size_t(query) * a.q_row;
            for (uint32_t e = lane; e < wide; e += 64) {
                const uint32_t h = e / a.dim;
                out[h * a.q_head + (e - h * a.dim)] = 0.f;
            }
        }
    }
}

__device__ inline bool finite(float x) { return fabsf(x) < INFINITY; }
// The three values that a weight of zero does not cancel; is(k, x): x is the k-th.
__device__ inline float special(int k) { return k == 0 ? INFINITY : k == 1 ? -INFINITY : NAN; }
__device__ inline float is(int k, float x) { return (k == 2 ? x != x : x == special(k)) ? 1.f : 0.f; }

// Floats of a row in a run's slots.
template <int DP>
constexpr int kSlotRow = DP <= 64 ? 64 : 128;

// What joining the four waves' sums of a row takes.
struct RowPlan {
    f32x4 weights;  // of the waves
    size_t at;      // its first dim in the outputs, or in the run's slot
    bool sees;      // any key
    bool sound;     // its weights are numbers
};
// The `rows` sums of row block rb of (sequence b, kv head) as the four waves by keys left
// them in LDS, joined: outputs where the run holds the `whole` unit, else means, maximum
// and weight to the run's slot (a unit's first run had it last, the others first). Sums meet
// weights that are divided already, so that FP32 holds what it holds of each wave's. The
// block's threads do it together; `plans` is LDS. odd[wave] becomes 1 where the wave met an
// output that is not finite, of weights that are numbers.
template <int DP, int RB, bool VEC>
__device__ inline void finish(const PagedArgs &a, uint32_t run, uint32_t b, uint32_t kv, uint32_t rb, uint32_t rows,
                              bool whole, bool starts, const float (&part)[kWaves][RB][DP + 4],
                              const float2 (&ml)[kWaves][RB], RowPlan (&plans)[RB], uint32_t (&odd)[kWaves]) {
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // nothing below is computed ahead of a caller's main loop
    if (tid < rows) {
        float most = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = fmaxf(most, ml[w][tid].x);
        const float from = most == -INFINITY ? 0.f : most;
        RowPlan p;
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            p.weights[w] = __builtin_amdgcn_exp2f(ml[w][tid].x - from);
            l = fmaf(p.weights[w], ml[w][tid].y, l);
        }
        p.sees = l != 0.f;
        p.sound = finite(l);
        p.weights *= 1.f / l;
        if (whole) {
            p.at = row_at(a, b, kv, rb * RB + tid);
        } else {
            const size_t slot = (2 * size_t(run) + starts) * RB + tid;
            p.at = slot * kSlotRow<DP>;
            reinterpret_cast<float2 *>(a.partial + 2 * size_t(a.runs) * RB * kSlotRow<DP>)[slot] = float2{most, l};
        }
        plans[tid] = p;
    }
    __syncthreads();
    float *const to = whole ? a.out : a.partial;
    float met = 0.f;  // NaN from an output on that is not finite
    for (uint32_t at = tid; at < rows * (DP / 4); at += kThreads) {
        const uint32_t row = at / (DP / 4), d = at % (DP / 4) * 4;
        const RowPlan &p = plans[row];
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) o += p.weights[w] * *reinterpret_cast<const f32x4 *>(&part[w][row][d]);
        if (!p.sees) o = f32x4{0.f, 0.f, 0.f, 0.f};  // a row that sees no key
        float all = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) all = VEC || d + e < a.dim ? fmaf(o[e], 0.f, all) : all;
        if (p.sound) met += all;
        if (VEC || !whole) {
            if (!whole || d < a.dim) *reinterpret_cast<f32x4 *>(to + p.at + d) = o;
        } else {
            store_dims<false>(to + p.at, int(d), int(a.dim), o);
        }
    }
    if (met != 0.f) odd[tid / 64] = 1;
}

// The outputs, or means in slots, of the block's run that this wave left and that are not
// finite, once more: those whose sums alone passed FP32's largest (values of 1e37 over a hundred
// equal keys) are finite then. A wave leaves OWN neighbouring rows of a unit, then its next.
// Weights are 2^-32 as large, which 2^24 keys of 1 each leave room for, and a row's
// values are summed by themselves: 64 keys' scores, a lane each, then their values, a lane for two
// dims. Not made to be fast, nor called where all is finite; and where the values themselves are
// not, that is found by one look at them (512 queries over 16384 keys of 128 dims, every 1024th
// value infinite: 5.5 ms, 3.5 without this). Inlined, as args_now() asks.
template <int TILE, int RB, int ROW, int OWN, bool VEC>
__device__ __attribute__((always_inline)) inline void sum_again() {
    constexpr uint32_t kPiece = 4096;  // keys whose sums are put aside
    __threadfence_block();  // other lanes left what this one looks at
    const PagedArgs &a = *(const PagedArgs *)args_now();  // no register keeps them for this across a main loop
    const Work<TILE, RB> work(a);
    const uint32_t run = run_of(blockIdx.x, a.runs);
    const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), waves = blockDim.x / 64;
    const uint32_t chunk = (work.total + a.runs - 1) / a.runs;
    uint32_t b, before;
    const uint32_t t_stop = work.start(run + 1, chunk, b, before);
    uint32_t t = work.start(run, chunk, b, before);
    while (t < t_stop) {
        const Sequence s = work.anew(b);
        if (!work.active(s)) {
            ++b;
            continue;
        }
        const uint32_t all = uniform(work.all_of(s));
        const Spot p = work.spot(s, all, t - before);
        const uint32_t begin = p.tile, end = min(p.tiles, begin + (t_stop - t));
        const bool whole = begin == 0 && end == p.tiles;
        const uint32_t rows = min(uint32_t(RB), s.count * a.group - p.rb * RB);
        const bool near = lane < a.dim, far = lane + 64 < a.dim;
        // The first token whose value is not finite, of this lane's dims; looked for where a row asks.
        uint32_t near_first = 0, far_first = 0;
        bool looked = false;
        for (uint32_t r = 0; r < rows; ++r) {
            if (r / OWN % waves != wave) continue;
            const uint32_t row = p.rb * RB + r;
            const size_t q_at = row_at(a, b, p.kv, row), slot = (2 * size_t(run) + (begin == 0)) * RB + r;
            float *const to = whole ? a.out + q_at : a.partial + slot * ROW;
            bool near_odd = near && !finite(to[lane]), far_odd = far && !finite(to[lane + 64]);
            if (!__any(near_odd || far_odd)) continue;
            if (!looked) {
                looked = true;
                near_first = far_first = ~0u;
                const uint32_t tokens = min(end * TILE, s.length);
                for (uint32_t key = begin * TILE; key < tokens; key += 16) {
                    const Place of = place_of(a, key / 16);
                    const uint32_t page = uniform(page_of(a, a.tables[size_t(b) * a.table + of.entry]));
                    if (page == kNoPage) continue;
                    const float *const v = a.v + page * a.p_page + p.kv * a.p_head + size_t(of.step) * 16 * a.p_row;
#pragma unroll 4
                    for (uint32_t i = 0; i < 16; ++i) {
                        const bool there = key + i < tokens;
                        const float x = there && near ? v[i * a.p_row + lane] : 0.f, y = there && far ? v[i * a.p_row + lane + 64] : 0.f;
                        if (!finite(x)) near_first = min(near_first, key + i);
                        if (!finite(y)) far_first = min(far_first, key + i);
                    }
                }
            }
            const int token = int(s.length) - int(s.count) + int(row / a.group);
            const uint32_t stop = token < 0 ? 0u : min(min(end * TILE, s.length), uint32_t(token) + 1);
            near_odd = near_odd && near_first >= stop;
            far_odd = far_odd && far_first >= stop;
            if (!__any(near_odd || far_odd)) continue;
            // A key's score, -inf where there is none; and its place in the pools.
            auto score_of = [&](uint32_t key, size_t &place) __attribute__((always_inline)) {
                const Place of = place_of(a, key / 16);
                const uint32_t page = key < stop ? page_of(a, a.tables[size_t(b) * a.table + of.entry]) : kNoPage;
                if (page == kNoPage) return -INFINITY;
                place = page * a.p_page + p.kv * a.p_head + (size_t(of.step) * 16 + key % 16) * a.p_row;
                float x = 0.f;
                for (uint32_t d = 0; d < a.dim; d += 4) {
                    const f32x4 q = load_dims<VEC>(a.q + q_at, int(d), int(a.dim)) * a.qscale;
                    const f32x4 k = load_dims<VEC>(a.k + place, int(d), int(a.dim));
#pragma unroll
                    for (int e = 0; e < 4; ++e) x = fmaf(q[e], k[e], x);
                }
                return x;
            };
            size_t place = 0;
            float top = -INFINITY;
            bool nan = false;
            for (uint32_t key = begin * TILE; key < stop; key += 64) {
                const float score = score_of(key + lane, place);
                top = fmaxf(top, score);
                nan |= score != score;
            }
#pragma unroll
            for (int d = 32; d; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
            if (!finite(top) || __any(nan)) continue;
            float sum = 0.f, sum_now = 0.f;
            float2 out = {0.f, 0.f}, now = out;
            for (uint32_t key = begin * TILE; key < stop; key += 64) {
                const float weight = __builtin_amdgcn_exp2f(score_of(key + lane, place) - top);
                sum_now += weight;
                for (uint32_t i = 0; i < min(64u, stop - key); ++i) {
                    const float w = __uint_as_float(of_lane(__float_as_uint(weight), int(i)));
                    if (w == 0.f) continue;
                    const size_t at = size_t(of_lane(uint32_t(place >> 32), int(i))) << 32 | of_lane(uint32_t(place), int(i));
                    if (near) now.x = fmaf(w * 0x1p-32f, a.v[at + lane], now.x);
                    if (far) now.y = fmaf(w * 0x1p-32f, a.v[at + lane + 64], now.y);
                }
                if ((key / 64 + 1) % (kPiece / 64) == 0 || key + 64 >= stop) {
                    sum += sum_now;
                    out.x += now.x;
                    out.y += now.y;
                    sum_now = now.x = now.y = 0.f;
                }
            }
#pragma unroll
            for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
            const float by = 0x1p32f / sum;
            if (near_odd) to[lane] = out.x * by;
            if (far_odd) to[lane + 64] = out.y * by;
        }
        t += end - begin;
        if (t >= before + all) {
            before += all;
            ++b;
        }
    }
}

}  // namespace paged
}  // namespace
}  // namespace hipk
}  // namespace jade
