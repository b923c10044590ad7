// Device parts shared by the ragged attention kernels: where a run's tiles lie, and
// how a row's sums become outputs or go to the workspace.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "attention_ragged.hpp"
#include "spec.hpp"
#include "whole.hpp"

namespace jade {
namespace hipk {
namespace {
namespace ragged {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;
constexpr uint32_t kCus = 256;
constexpr float kLazyMax = 8.0f;   // log2 units: the running maximum moves only past this
constexpr uint32_t kRawBuffer = 0x00020000;    // buffer descriptor word 3: raw buffer, 32-bit data format
constexpr uint32_t kDeadOffset = 0x80000000u;  // past every tile: reads zero
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kWords = int(kMaxTreeNodes) / 64;

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

// The tiles of every sequence, of one (kv head, row block) each. A lane has the
// sequences of its number modulo 64; those of the first 64 stay in registers, so that
// one load of the lengths is all that the first loads of keys wait for.
template <int TILE>
struct Spread {
    const RaggedArgs &a;
    const uint32_t draft_tiles, len, own, up_to;  // of sequence (lane): length, tiles, tiles up to it
    uint32_t total;

    __device__ uint32_t load_length(uint32_t b) const { return b < a.batch ? whole_below(a.lengths[b], a.keys) : 0u; }
    __device__ uint32_t tiles_of(uint32_t b, uint32_t length) const {
        return b < a.batch ? (length + TILE - 1) / TILE + draft_tiles : 0u;
    }
    // Of one sequence, for the whole wave.
    __device__ uint32_t length(uint32_t b) const { return b < 64 ? of_lane(len, int(b)) : uniform(load_length(b)); }
    __device__ uint32_t tiles_at(uint32_t b) const { return tiles_of(b, length(b)); }
    __device__ explicit Spread(const RaggedArgs &args)
        : a(args), draft_tiles((a.nodes + TILE - 1) / TILE), len(load_length(threadIdx.x & 63)),
          own(tiles_of(threadIdx.x & 63, len)), up_to(scan_add(own)), total(of_lane(up_to, 63)) {
        for (uint32_t b0 = 64; b0 < a.batch; b0 += 64) total += of_lane(scan_add(lane_tiles(b0)), 63);
    }
    // This lane's tiles among the sequences from b0 on.
    __device__ uint32_t lane_tiles(uint32_t b0) const {
        const uint32_t b = b0 + (threadIdx.x & 63);
        return tiles_of(b, load_length(b));
    }
    // The sequence that tile t < total belongs to, and the tiles before it.
    __device__ void find(uint32_t t, uint32_t &b, uint32_t &before) const {
        before = 0;
        uint32_t sum = up_to, mine = own;
        for (b = 0;; b += 64, mine = lane_tiles(b), sum = scan_add(mine)) {
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
    // block) where a run has four or more whole ones of that sequence: then none of them
    // needs joining, and runs with neighbouring row blocks, which read the same keys, do so
    // at the same time, from their XCD's L2 (4 x 32 heads x 1000 queries x 4096 keys: 1540
    // us with every run as long as the next, 1503 so). `b` and `before` as find() leaves
    // them; at the last tile's end they say nothing.
    __device__ uint32_t start(uint32_t run, uint32_t chunk, uint32_t units, uint32_t &b, uint32_t &before) const {
        const uint64_t at = uint64_t(run) * chunk, end = uint64_t(total) * units;
        if (at >= end) return uint32_t(end);
        uint32_t t = uint32_t(at);
        find(t / units, b, before);
        const uint32_t tiles = tiles_at(b);
        if (!rounds(tiles, chunk)) return t;
        const uint32_t over = (t - before * units) % tiles;
        t = 2 * over < tiles ? t - over : t - over + tiles;
        if (t == (before + tiles) * units) {
            before += tiles;
            ++b;
        }
        return t;
    }
    __device__ static bool rounds(uint32_t tiles, uint32_t chunk) { return 4 * tiles <= chunk; }
    // The tiles before sequence b.
    __device__ uint32_t before(uint32_t b) const {
        uint32_t sum = 0, last = up_to - own;
        for (uint32_t b0 = 64; b0 <= b; b0 += 64) {
            sum += b0 == 64 ? of_lane(up_to, 63) : of_lane(scan_add(lane_tiles(b0 - 64)), 63);
            const uint32_t mine = lane_tiles(b0);
            last = scan_add(mine) - mine;
        }
        return sum + of_lane(last, int(b & 63));
    }
};

__device__ inline bool is_node(float parent, int n) {
    return parent == -1.f || (parent >= 0.f && parent < float(n) && parent == truncf(parent));
}

// Run of block `id`: the runs of one XCD are neighbours.
__device__ inline uint32_t run_of(uint32_t id, uint32_t runs) { return id % 8 * (runs / 8) + id / 8; }

__device__ inline float across_keys_max(float x) {
    return fmaxf(fmaxf(x, __shfl_xor(x, 16)), fmaxf(__shfl_xor(x, 32), __shfl_xor(x, 48)));
}
__device__ inline float across_keys_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// Dims d .. d + 3 of a row, zeros from `dim` on and for no row. VEC: dim % 4 == 0 and
// 16-byte rows. Asked at run time its branches cost 1.2 us a launch (8 heads x 1024 keys of
// 64 dims, one query: 9.9 against 8.7 us).
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
// Row r of (sequence b, kv head): its sums o of dims d .. d + 3 over its weights' sum.
template <bool VEC>
__device__ inline void store_row(const RaggedArgs &a, uint32_t b, uint32_t kv, uint32_t r, uint32_t d, f32x4 o, float l) {
    const uint32_t head = r / a.queries, query = r - head * a.queries;
    const bool node = !a.nodes || is_node(a.parents[size_t(b) * a.nodes + query], int(query));
    o = node ? o * (1.0f / l) : f32x4{0.f, 0.f, 0.f, 0.f};
    float *const row = a.out + size_t(b) * a.q_batch + (size_t(kv) * a.group + head) * a.q_head + size_t(query) * a.q_row;
    store_dims<VEC>(row, int(d), int(a.dim), o);
}

__device__ inline bool finite(float x) { return fabsf(x) < INFINITY; }

// Floats of a row in a run's slots.
template <int DP>
constexpr int kSlotRow = DP <= 64 ? 64 : 128;

// What joining the four waves' sums of a row takes.
struct RowPlan {
    f32x4 weights;  // of the waves, with the whole sum's reciprocal where the row is finished
    float2 top_sum;
    size_t at;  // its first dim in the outputs, or in the run's slot
};
// A unit's sums as its four waves by keys left them in LDS, joined: outputs where the
// run holds the `whole` unit, else sums, maximum and weight to the run's slot (a unit's
// first run had it last, the others first). The block's threads do it together; `plans`
// is LDS. The sums in LDS are to be multiplied by `unscale`. True for a thread that met one
// that is not finite.
template <int DP, int RB, bool VEC>
__device__ inline bool finish(const RaggedArgs &a, uint32_t run, uint32_t b, uint32_t kv, uint32_t rb, bool whole,
                              bool starts, const float (&part)[kWaves][RB][DP + 4], const float2 (&ml)[kWaves][RB],
                              RowPlan (&plans)[RB], const uint64_t (&sees)[kMaxTreeNodes][kWords], float unscale) {
    const uint32_t rows = min(uint32_t(RB), a.group * a.queries - rb * RB);
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
        p.top_sum = float2{most, l};
        if (whole) {
            const uint32_t r = rb * RB + tid, head = r / a.queries, query = r - head * a.queries;
            p.at = size_t(b) * a.q_batch + (size_t(kv) * a.group + head) * a.q_head + size_t(query) * a.q_row;
            // A whole unit has the tree's tiles, and with them who sees whom.
            p.top_sum.y = a.nodes && !(sees[query][query / 64] >> (query & 63) & 1) ? 0.f : unscale / l;
        } else {
            const size_t slot = (2 * size_t(run) + starts) * RB + tid;
            p.at = slot * kSlotRow<DP>;
            reinterpret_cast<float2 *>(a.partial + 2 * size_t(a.runs) * RB * kSlotRow<DP>)[slot] = p.top_sum;
            p.top_sum.y = unscale;
        }
        plans[tid] = p;
    }
    __syncthreads();
    float *const to = whole ? a.out : a.partial;
    bool odd = false;
    for (uint32_t at = tid; at < rows * (DP / 4); at += kThreads) {
        const uint32_t row = at / (DP / 4), d = at % (DP / 4) * 4;
        const RowPlan &p = plans[row];
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) o += p.weights[w] * *reinterpret_cast<const f32x4 *>(&part[w][row][d]);
        if (p.top_sum.y != 0.f && d < uint32_t(a.dim))
#pragma unroll
            for (int e = 0; e < 4; ++e)
                odd |= (VEC || d + e < uint32_t(a.dim)) && !finite(o[e]);
        // A slot without a node is zeros whatever its sums are.
        o = p.top_sum.y == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o * p.top_sum.y;
        if (VEC || !whole) {
            if (!whole || d < uint32_t(a.dim)) *reinterpret_cast<f32x4 *>(to + p.at + d) = o;
        } else {
            store_dims<false>(to + p.at, int(d), int(a.dim), o);
        }
    }
    return odd;
}

// The tree of sequence b in LDS, by all threads of the block (each with the parent
// `mine` of slot threadIdx.x): bit n' of row n where node n sees node n'. Ancestors by
// doubling: after k steps a node has those up to 2^k above it.
__device__ inline void see_ancestors(uint32_t nodes, float mine, uint64_t (&sees)[kMaxTreeNodes][kWords],
                                     int (&above)[kMaxTreeNodes]) {
    __syncthreads();
    const int n = threadIdx.x;
    int parent = -2;
    if (nodes <= 64) {  // one wave by itself, without barriers (28 nodes: 32.0 us of a launch by all, 29.9 so)
        if (n < 64) {
            if (n < int(nodes)) parent = is_node(mine, n) ? int(mine) : -2;
            uint32_t lo = parent != -2 && n < 32 ? 1u << n : 0u, hi = parent != -2 && n >= 32 ? 1u << (n - 32) : 0u;
            for (uint32_t reach = 1; reach < nodes; reach *= 2) {
                const int from = max(parent, 0);
                const uint32_t more_lo = __shfl(lo, from), more_hi = __shfl(hi, from);
                const int next = __shfl(parent, from);
                if (parent >= 0) {
                    lo |= more_lo;
                    hi |= more_hi;
                    parent = next;
                }
            }
            sees[n][0] = uint64_t(hi) << 32 | lo;
            sees[n][1] = 0;
        }
        __syncthreads();
        return;
    }
    if (n < int(nodes)) {
        parent = is_node(mine, n) ? int(mine) : -2;
        above[n] = parent;
#pragma unroll
        for (int w = 0; w < kWords; ++w) sees[n][w] = parent != -2 && n / 64 == w ? 1ull << (n & 63) : 0ull;
    }
    for (uint32_t reach = 1; reach < nodes; reach *= 2) {
        __syncthreads();
        uint64_t more[kWords] = {};
        int next = parent;
        if (parent >= 0) {
#pragma unroll
            for (int w = 0; w < kWords; ++w) more[w] = sees[parent][w];
            next = above[parent];
        }
        __syncthreads();
        if (parent >= 0) {
#pragma unroll
            for (int w = 0; w < kWords; ++w) sees[n][w] |= more[w];
            above[n] = parent = next;
        }
    }
    __syncthreads();
}

// The three values that a weight of zero does not cancel; is(k, x): x is the k-th.
__device__ inline float special(int k) { return k == 0 ? INFINITY : k == 1 ? -INFINITY : NAN; }
__device__ inline float is(int k, float x) { return (k == 2 ? x != x : x == special(k)) ? 1.f : 0.f; }

}  // namespace ragged
}  // namespace
}  // namespace hipk
}  // namespace jade
