// Attention of a chunk of new tokens of every sequence over its pages
// (attention_paged); one new token is ordinary decoding. Token j of sequence b is row
// j % page of page tables[b, j / page]; query i < counts[b] is token
// lengths[b] - counts[b] + i and sees the tokens up to itself:
//   out_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i), s_ij = q_i k_j / sqrt(dim).
// Queries past a sequence's count, and those that see no key, are zeros. An entry of a table
// that names no page is 16 or more tokens that nobody sees.
//
// The kernel of attention_ragged.hip over pages: one pass with a running maximum and sum,
// FP32 MFMAs (16x16x4) in the transposed form, K, V and P in registers, four waves that take
// 16 keys each of a tile of 64. Pages hold multiples of 16 tokens, so that a wave's 16 keys
// lie in one page, whose row of the table it looks up a tile ahead; each has a descriptor of
// its own, which ends with the sequence's last token, so no offset passes 2^31 however large
// the pool, and what lies past the last token or in no page reads as zeros.
//
// All tiles of all (sequence, kv head, row block)s in a row are cut into equal runs, one a
// block; a launch of its own joins what a cut went through.
//
// Up to 16 rows it is bound by reading K and V: 16 sequences of 4096 to 8192 keys, 32 heads (8
// of keys) of 128, one query each, 834 MB in pages of 16 tokens: 145 us, 5.7 TB/s, and 4.6 us
// for the join. One sequence of 1000 keys, 8 heads of 64: 7.1 and 4.2 us, each a chain of
// loads that wait for one another (lengths, table, keys; lengths, sums). Many sequences of few
// keys are bound by what a unit takes from its first load to its outputs: 1024 of 50 to 100
// keys, 8 kv heads of 128, 629 MB in 175 us. Besides, every wave walks the whole batch, 64
// sequences at a time, before it knows its run.
#include <cmath>

#include "attention_paged.hpp"
#include "kernels.hpp"

namespace jade {
namespace hipk {
namespace {

using namespace paged;

constexpr int kTile = 64;  // keys of a tile
// Tiles after which a wave's sums are put aside and begun anew: FP32 sums of 65536 equal
// weights each were off by up to 2.9e-3 (512 sequences of 2^20 tokens, one run each).
constexpr uint32_t kPiece = 64;

// DP: head dim padded (64, 96, 128). G: groups of 16 rows, all of them every wave's.
template <int DP, int G>
constexpr int kWavesASimd = DP > 64 && G == 2 ? 1 : 2;  // what the registers hold
template <int DP, int G, bool VEC>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(kWavesASimd<DP, G>, kWavesASimd<DP, G>))) void attention_paged(PagedArgs a) {
    constexpr int KJ = DP / 16, NJ = (DP + 63) / 64, RB = 16 * G, OUT = 64 * NJ;
    __shared__ __attribute__((aligned(16))) float part[kWaves][RB][OUT + 4];
    __shared__ float2 ml[kWaves][RB];
    __shared__ RowPlan plans[RB];
    __shared__ uint32_t odd_outputs[kWaves];  // whether a wave met an output that is not finite
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = uniform(tid >> 6);
    odd_outputs[wave] = 0;
    const int m = lane & 15, g = lane >> 4;
    const Work<kTile, RB> work(a);
    const uint32_t chunk = (work.total + a.runs - 1) / a.runs;
    const uint32_t run = run_of(blockIdx.x, a.runs);
    uint32_t b, before;
    const uint32_t t_stop = work.start(run + 1, chunk, b, before);
    uint32_t t = work.start(run, chunk, b, before);

    const uint32_t row_bytes = a.p_row * 4u;
    uint32_t koff[KJ], voff[NJ][4];
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
        const uint32_t d = 16 * j + 4 * g;
        koff[j] = d < a.dim ? uint32_t(m) * row_bytes + d * 4u : kDeadOffset;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t d = 64 * j + 4 * m;
            voff[j][i] = d < a.dim ? uint32_t(4 * g + i) * row_bytes + d * 4u : kDeadOffset;
        }

    // The part of a (sequence, kv head, row block) that tile t of the launch begins in this
    // run; nothing where the run is over. Tiles from `stop` on show its rows nothing.
    struct Unit {
        uint32_t b, before, kv, rb, begin, end, stop, tiles, all;
        Sequence s;
    };
    auto unit_at = [&](uint32_t t, uint32_t b, uint32_t before) {
        Unit u{};
        if (t >= t_stop) return u;
        for (u.b = b, u.before = before;; ++u.b) {  // the run ends with a sequence that has tiles
            u.s = work.at(u.b);
            if (work.active(u.s)) break;
        }
        u.all = work.all_at(u.b, u.s);
        const Spot p = work.spot(u.s, u.all, t - u.before);
        u.kv = p.kv;
        u.rb = p.rb;
        u.begin = p.tile;
        u.tiles = p.tiles;
        u.end = min(u.tiles, u.begin + (t_stop - t));
        const int last = int(u.s.length) - int(u.s.count) + int(min(u.s.count - 1, (u.rb * RB + RB - 1) / a.group));
        u.stop = last < 0 ? 0u : u.end;
        return u;
    };
    // The table's entry for this wave's keys of tile x, -1 past `stop`.
    auto entry_of = [&](const Unit &u, uint32_t x) {
        const uint32_t n = x * (kTile / 16) + wave;
        return x < u.stop && n * 16 < u.s.length ? a.tables[size_t(u.b) * a.table + place_of(a, n).entry] : -1.f;
    };
    // Those keys or values: zeros where they have no page.
    auto tile_of = [&](const float *pool, const Unit &u, uint32_t x, uint32_t page) {
        const uint32_t n = x * (kTile / 16) + wave;
        const bool some = page != kNoPage;
        const float *from = pool + (some ? page * a.p_page + u.kv * a.p_head + size_t(place_of(a, n).step) * 16 * a.p_row : 0);
        const uint32_t bytes = some ? (min(u.s.length - n * 16, 16u) - 1) * row_bytes + a.dim * 4u : 0u;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(from), 0, int(bytes), int(kRawBuffer));
    };
    // A last chunk that is not whole reads into the next row, or nothing past the tile.
    auto load = [&](__amdgpu_buffer_rsrc_t from, uint32_t at) {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, int(at), 0, 0));
    };
    f32x4 kf[KJ], vf[NJ][4], qf[G][KJ];
    auto load_k = [&](const Unit &u, uint32_t x, uint32_t page) {
        const auto from = tile_of(a.k, u, x, page);
#pragma unroll
        for (int j = 0; j < KJ; ++j) kf[j] = load(from, koff[j]);
    };
    auto load_v = [&](const Unit &u, uint32_t x, uint32_t page) {
        const auto from = tile_of(a.v, u, x, page);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) vf[j][i] = load(from, voff[j][i]);
    };
    auto rows_of = [&](const Unit &u) { return min(uint32_t(RB), u.s.count * a.group - u.rb * RB); };
    // Q^T operand: row 16 r + m of the block, dims 16 j + 4 g + e.
    auto load_rows = [&](const Unit &u) {
        if (u.begin == u.end) return;
#pragma unroll
        for (int r = 0; r < G; ++r) {
            const float *row = 16 * r + m < rows_of(u) ? a.q + row_at(a, u.b, u.kv, u.rb * RB + 16 * r + m) : nullptr;
#pragma unroll
            for (int j = 0; j < KJ; ++j) qf[r][j] = load_dims<VEC>(row, 16 * j + 4 * g, a.dim);
        }
    };
    auto page_at = [&](float entry) { return uniform(page_of(a, entry)); };
    Unit u = unit_at(t, b, before);
    uint32_t page = page_at(entry_of(u, u.begin));  // of the tile at hand
    float ahead = entry_of(u, u.begin + 1);         // of the one after
    load_k(u, u.begin, page);
    load_v(u, u.begin, page);
    load_rows(u);
    while (u.begin < u.end) {
        const uint32_t begin = u.begin;
        const bool whole = begin == 0 && u.end == u.tiles;
        // The unit after this one, whose first loads go beside this one's last products.
        t += u.end - begin;
        const bool over = t >= u.before + u.all;
        const Unit next = unit_at(t, u.b + over, over ? u.before + u.all : u.before);
        const float first = entry_of(next, next.begin), second = entry_of(next, next.begin + 1);
#pragma unroll
        for (int r = 0; r < G; ++r)
#pragma unroll
            for (int j = 0; j < KJ; ++j) qf[r][j] *= a.qscale;  // log2 units

        f32x4 acc[G][NJ][4];
        float top[G], sum[G];
#pragma unroll
        for (int r = 0; r < G; ++r) {
            top[r] = -INFINITY;
            sum[r] = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][j][e] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        // Tokens of the block's first query and of this lane's rows.
        const int old = int(u.s.length) - int(u.s.count), low = old + int(u.rb * RB / a.group);
        int mine[G];
#pragma unroll
        for (int r = 0; r < G; ++r) mine[r] = old + int((u.rb * RB + 16 * r + m) / a.group);
        uint32_t page_next = page;
        if (begin >= u.stop) {  // no tile of this unit's: the next one's
            page_next = page_at(first);
            load_k(next, next.begin, page_next);
            load_v(next, next.begin, page_next);
        }
        // This wave's sums since the last time, on top of those, in LDS: row 16 r + m, dims
        // 64 j + 16 g + 4 i + e.
        auto put_aside = [&](bool first) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < G; ++r) {
                float2 &kept = ml[wave][16 * r + m];
                const float2 old = first ? float2{-INFINITY, 0.f} : kept;
                const float all = across_keys_sum(sum[r]), from = top[r] == -INFINITY ? 0.f : top[r];
                const float weight = __builtin_amdgcn_exp2f(old.x - from);
                if (g == 0) kept = float2{top[r], fmaf(weight, old.y, all)};
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        f32x4 &to = *reinterpret_cast<f32x4 *>(&part[wave][16 * r + m][64 * j + 16 * g + 4 * i]);
                        const f32x4 x = {acc[r][j][0][i], acc[r][j][1][i], acc[r][j][2][i], acc[r][j][3][i]};
                        to = first ? x : x + weight * to;
                    }
            }
        };
        for (uint32_t x = begin; x < u.stop; ++x) {
            const bool last = x + 1 == u.stop;
            if (x != begin && (x - begin) % kPiece == 0) {
                if (x - begin == kPiece) __syncthreads();  // the last unit's sums are read
                put_aside(x - begin == kPiece);
#pragma unroll
                for (int r = 0; r < G; ++r) {
                    sum[r] = 0.f;
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[r][j][e] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
            }
            if (!VEC)  // the next row's values may not be finite
#pragma unroll
                for (int j = 0; j < KJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (16 * j + 4 * g + e >= a.dim) kf[j][e] = 0.f;
            f32x4 p[G] = {};  // scores, then weights, of keys 16 wave + 4 g + i
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int r = 0; r < G; ++r)
                        p[r] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][e], qf[r][j][e], p[r], 0, 0, 0);
            page_next = page_at(last ? first : ahead);
            last ? load_k(next, next.begin, page_next) : load_k(u, x + 1, page_next);
            ahead = entry_of(u, x + 2);
            const bool masked = int(x * kTile + kTile) > low + 1;
            if (masked || page == kNoPage) {
                const int key = int(x) * kTile + 16 * int(wave) + 4 * g;
#pragma unroll
                for (int r = 0; r < G; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key + i > mine[r] || page == kNoPage) p[r][i] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < G; ++r) {
                const float most = fmaxf(fmaxf(p[r].x, p[r].y), fmaxf(p[r].z, p[r].w));
                if (__any(most > top[r] + kLazyMax)) {
                    const float reached = fmaxf(top[r], across_keys_max(most));
                    const float keep = reached == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top[r] - reached);
                    top[r] = reached;
                    sum[r] *= keep;
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[r][j][e] *= keep;
                }
                const float from = top[r] == -INFINITY ? 0.f : top[r];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[r][i] = __builtin_amdgcn_exp2f(p[r][i] - from);
                    sum[r] += p[r][i];
                }
            }
            bool odd = false;
            if (masked && u.s.count > 1) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) odd |= !finite(vf[j][i][e]);
            }
            if (!__any(odd)) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int r = 0; r < G; ++r)
                                acc[r][j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[j][i][e], p[r][i], acc[r][j][e], 0, 0, 0);
            } else {
                // A value that is not finite, of a token that not every row may see: the
                // finite ones, then the weight that each row gives to each special one.
#pragma unroll
                for (int r = 0; r < G; ++r)
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int k = -1; k < 3; ++k) {
                                __builtin_amdgcn_sched_barrier(0);  // one at a time: a rare path takes no registers
                                f32x4 sums = k < 0 ? acc[r][j][e] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float v = vf[j][i][e], y = k >= 0 ? is(k, v) : finite(v) ? v : 0.f;
                                    sums = __builtin_amdgcn_mfma_f32_16x16x4f32(y, p[r][i], sums, 0, 0, 0);
                                }
                                if (k < 0)
                                    acc[r][j][e] = sums;
                                else
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        if (sums[i] > 0.f) acc[r][j][e][i] += special(k);
                            }
            }
            last ? load_v(next, next.begin, page_next) : load_v(u, x + 1, page_next);
            page = page_next;
        }
        page = page_next;
        ahead = second;
        const uint32_t rows = rows_of(u);
        load_rows(next);

        // The four waves' sums joined.
        __syncthreads();
        put_aside(u.stop <= begin + kPiece);
        __syncthreads();
        finish<OUT, RB, VEC>(a, run, u.b, u.kv, u.rb, rows, whole, begin == 0, part, ml, plans, odd_outputs);
        u = next;
    }
    clear_rows(work);
    if (__builtin_expect(uniform(odd_outputs[wave]), 0)) sum_again<kTile, RB, OUT, kThreads / OUT, VEC>();
}

// How the launch that joins is laid out: blocks x rows, and which unit a block has.
struct JoinGrid {
    uint32_t x, y;
    bool shared, by_unit;
};

// What the runs left of a (sequence, kv head, row block) cut between them: block x has unit
// x (BY_UNIT), or the unit that the cut before run x + 1 is the first of. DP / 4 lanes have a
// row; ROWS rows of a unit go to a block, each with all of its slots, or (ROWS 1) one, with
// the slots shared out (a unit of many runs).
template <int DP, int RB, int TILE, int ROWS, bool BY_UNIT, bool VEC>
__device__ void join_unit(const PagedArgs &a, uint32_t block, uint32_t rows_from) {
    constexpr int LANES = DP / 4, PARTS = kThreads / LANES / ROWS;
    __shared__ __attribute__((aligned(16))) f32x4 sums[PARTS][LANES];
    __shared__ float2 weights[PARTS];
    const int tid = threadIdx.x, lane = tid % LANES, p = ROWS == 1 ? tid / LANES : 0;
    const uint32_t row = rows_from * ROWS + (ROWS == 1 ? 0 : tid / LANES), d = 4 * lane;
    const Work<TILE, RB> work(a);
    const uint32_t chunk = (work.total + a.runs - 1) / a.runs;
    uint32_t b, before, unit, cut = 0;
    if (BY_UNIT) {
        if (!work.find_unit(block, b, unit, before)) return;
    } else {
        cut = work.start(block + 1, chunk, b, before);
        if (cut == work.total) return;
    }
    const Sequence s = work.at(b);
    if (!work.active(s) || work.rounds(s, chunk)) return;  // at a sequence's start; whole units
    Spot at;
    uint32_t start;
    if (BY_UNIT) {
        const uint32_t blocks = work.blocks(s), head = work.all_at(b, s) / a.kv_heads;
        at.kv = unit / blocks;
        at.rb = unit - at.kv * blocks;
        at.tiles = work.tiles(s, at.rb);
        start = before + at.kv * head + work.tiles_before(s, at.rb);
    } else {
        at = work.spot(s, work.all_at(b, s), cut - before);
        start = cut - at.tile;
        if (start + chunk < cut || start == cut) return;  // not its first cut
    }
    const uint32_t kv = at.kv, rb = at.rb, tiles = at.tiles;
    const bool mine = row < min(uint32_t(RB), s.count * a.group - rb * RB);
    const uint32_t first = start / chunk, last = (start + tiles - 1) / chunk;
    if (first == last) return;
    const float2 *ml = reinterpret_cast<const float2 *>(a.partial + 2 * size_t(a.runs) * RB * DP);
    // A unit's first run had it last, the others first.
    auto slot = [&](uint32_t r) { return (2 * size_t(r) + (r == first)) * RB + row; };
    // The mean of the slots' means so far, weighed by their shares of the weight: no sum passes
    // the values. Four slots at a time, on their way together.
    constexpr int kAtOnce = 4;
    float most = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};  // zeros for a row that sees no key
    for (uint32_t r0 = first + p; mine && r0 <= last; r0 += kAtOnce * PARTS) {
        float2 x[kAtOnce];
        f32x4 means[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const uint32_t r = r0 + i * PARTS;
            x[i] = r <= last ? ml[slot(r)] : float2{-INFINITY, 0.f};
            means[i] = r <= last ? *reinterpret_cast<const f32x4 *>(a.partial + slot(r) * DP + d) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
        const float was = most;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) most = fmaxf(most, x[i].x);
        const float from = most == -INFINITY ? 0.f : most, old = l * __builtin_amdgcn_exp2f(was - from);
        l = old;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) l += x[i].y *= __builtin_amdgcn_exp2f(x[i].x - from);
        const float by = l == 0.f ? 0.f : 1.0f / l;
        o *= old * by;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) o += means[i] * (x[i].y * by);
    }
    if constexpr (PARTS > 1) {
        sums[p][lane] = o;
        if (lane == 0) weights[p] = float2{most, l};
        __syncthreads();
        if (p) return;
#pragma unroll
        for (int x = 1; x < PARTS; ++x) most = fmaxf(most, weights[x].x);
        const float from = most == -INFINITY ? 0.f : most;
        float shares[PARTS];
        l = 0.f;
#pragma unroll
        for (int x = 0; x < PARTS; ++x) l += shares[x] = weights[x].y * __builtin_amdgcn_exp2f(weights[x].x - from);
        const float by = l == 0.f ? 0.f : 1.0f / l;  // a row that sees no key is zeros
        o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < PARTS; ++x) o += sums[x][lane] * (shares[x] * by);
    }
    if (!mine) return;
    store_dims<VEC>(a.out + row_at(a, b, kv, rb * RB + row), int(d), int(a.dim), o);
}
template <int DP, int RB, int TILE, bool VEC>
__device__ void join(const PagedArgs &a, const JoinGrid &g, uint32_t block) {
    constexpr int kRowsOf = kThreads / (DP / 4);  // rows of a block
    const uint32_t y = block / g.x, x = block - y * g.x;
    if (g.shared)
        join_unit<DP, RB, TILE, 1, true, VEC>(a, x, y);
    else if (g.by_unit)
        join_unit<DP, RB, TILE, kRowsOf, true, VEC>(a, x, y);
    else
        join_unit<DP, RB, TILE, kRowsOf, false, VEC>(a, x, y);
}
// Both launches' units: of the one for few rows, then of the one for many.
template <int DP, int RB, bool VEC>
__global__ __launch_bounds__(kThreads) void attention_paged_join(PagedArgs few, JoinGrid few_grid, PagedArgs many,
                                                                 JoinGrid many_grid) {
    const uint32_t blocks = few_grid.x * few_grid.y;
    if (blockIdx.x < blocks)
        join<DP, RB, kTile, VEC>(few, few_grid, blockIdx.x);
    else if constexpr (VEC && RB == 16)
        join<DP, DP == 64 ? 128 : 256, int(kPagedFlashTile), VEC>(many, many_grid, blockIdx.x - blocks);
}

uint64_t rows_of(const PagedShape &s) { return uint64_t(s.heads / s.kv_heads) * s.queries; }

// Sequences of more rows than this, for each kv head, go to the kernel on bf16 parts
// (attention_paged_flash.hip), by a launch of its own. Measured, this kernel and that one, 8
// sequences of at most 4096 keys, 8 kv heads, 48 rows. In calls that have no others, by two groups
// here: dims of 32 55.0 and 51.5 us, of 40 55.8 and 60.0, of 64 57.4 and 60.9, of 80 96.8 and 87.5,
// of 96 98.9 and 90.2, of 128 108 and 101. In calls whose spec has more, by one: 48.4 and 52.7,
// 52.6 and 59.7, 64.2 and 62.4, 84.6 and 89.8, 87.8 and 92.4, 122 and 106. One sequence of 8192
// keys, dims of 64: 26.1 and 30.0, 27.3 and 32.5. 64 rows of 64 dims in a call that has more:
// 75.5 and 61.5.
uint32_t few_rows(const PagedShape &s) { return s.dim <= 64 ? 48 : 32; }
// That kernel takes whole float4s and offsets of a sequence's rows in 31 bits. What it does not
// take reads K and V again for every 32 rows here, and counts its tiles row block by row block
// before the first key is loaded: 512 queries, 32 heads (8 of keys), 8192 keys, dims of 37 400
// us (40 217), of 126 902 (128 358).
bool has_many(const PagedShape &s) {
    return s.dim % 4 == 0 && rows_of(s) > few_rows(s) && uint64_t(s.heads) * s.queries * s.dim < 1u << 29;
}

// One of the two launches: its rows a block; (sequence, kv head, row block)s and their tiles
// where all sequences are of full length.
struct Half {
    uint32_t rows, dims;  // dims of a row in a run's slots
    uint64_t units, tiles;
    uint32_t runs;
};
Half half_of(const PagedShape &s, uint64_t rows, uint32_t rb, uint32_t tile, uint32_t blocks) {
    Half x{rb, s.dim > 64 ? 128u : 64u, 0, 0, 0};
    x.units = uint64_t(s.batch) * s.kv_heads * ((rows + rb - 1) / rb);
    x.tiles = x.units * ((uint64_t(s.table) * s.page + tile - 1) / tile);
    // As many blocks as work on the chip at once, or one per tile where there can be no more.
    x.runs = x.tiles >= blocks ? blocks : uint32_t((x.tiles + 7) / 8 * 8);
    return x;
}
// Two groups of rows a wave, which read K and V once for both, where a kv head has more than
// one and none goes to the other launch (which leaves sequences of few new tokens to this
// one). 32 rows, one group and two: 8 sequences of at most 4096 keys, 8 kv heads of 64 42.1
// and 36.8 us, of 80 56.6 and 61.2 (57 since), of 128 80.3 and 62.2; one sequence of 8192 23.0
// and 20.1, 29.2 and 25.6, 34.0 and 28.3.
uint32_t groups_of(const PagedShape &s) { return rows_of(s) > 16 && !has_many(s) ? 2 : 1; }
Half few_of(const PagedShape &s) {
    const uint32_t groups = groups_of(s);
    return half_of(s, has_many(s) ? few_rows(s) : rows_of(s), 16 * groups, kTile, groups == 2 && s.dim > 64 ? kCus : 2 * kCus);
}
Half many_of(const PagedShape &s) {
    return half_of(s, rows_of(s), paged_flash_rows(s.dim), kPagedFlashTile, s.dim <= 64 ? 2 * kCus : kCus);
}
// Short caches: whole (sequence, kv head, row block)s to every run, and no launch that joins.
// Where none is longer than two tiles, or there are as many as runs and none is longer than
// four (eight on parts). Cut and joined, and whole: 8 heads of 64, one query, at most 64 keys
// 8.3 and 6.4 us, 128 9.2 and 7.3; 64 x 8 kv heads of 128, at most 128 17.8 and 15.8, 256 28.0 and
// 25.4; but 16 x 8, 256 keys 14.9 and 18.2; on parts 8 units of four tiles 13.7 and 15.5.
bool uncut(const PagedShape &s) {
    auto whole = [&](const Half &x, uint32_t most) {
        return x.tiles <= 2 * x.units || (x.units >= x.runs && x.tiles <= most * x.units);
    };
    return whole(few_of(s), 4) && (!has_many(s) || whole(many_of(s), 8));
}

size_t bytes_of(const Half &x) { return 2 * size_t(x.runs) * x.rows * (x.dims + 2) * sizeof(float); }

JoinGrid join_grid(const PagedShape &s, const Half &x) {
    const uint64_t all = rows_of(s);
    const uint32_t rows = all < x.rows ? uint32_t(all) : x.rows, rows_of_block = uint32_t(kThreads) / (x.dims / 4);
    // Units of 16 runs or more: their slots are shared out; else whole rows.
    const bool shared = 16 * x.units <= x.runs, by_unit = x.units < x.runs;
    return {by_unit ? uint32_t(x.units) : x.runs - 1, shared ? rows : (rows + rows_of_block - 1) / rows_of_block, shared, by_unit};
}

template <int DP, int G, bool VEC>
hipError_t launch(hipStream_t stream, const PagedShape &s, PagedArgs few, float *workspace) {
    static_assert(DP == kSlotRow<DP>, "slots are of 64 or 128 dims");
    const bool both = VEC && G == 1 && has_many(s);
    const Half half = few_of(s), other = many_of(s);
    PagedArgs many = few;
    few.least_rows = 1;
    few.most_rows = both ? few_rows(s) : ~0u;
    few.runs = half.runs;
    few.uncut = many.uncut = uncut(s);
    few.partial = workspace;
    const JoinGrid few_grid = join_grid(s, half);
    JoinGrid many_grid{1, 0, false, false};
    // Scores of 96 dims rather than 128: 32 rows over 8 sequences of at most 4096 keys, 8 kv
    // heads of 80, 56.8 -> 51.7 us; 16 x 24 heads, one row, at most 1531 keys 65.6 -> 63.4.
    if (DP == 128 && s.dim <= 96)
        hipLaunchKernelGGL((attention_paged<96, G, VEC>), dim3(few.runs), dim3(kThreads), 0, stream, few);
    else
        hipLaunchKernelGGL((attention_paged<DP, G, VEC>), dim3(few.runs), dim3(kThreads), 0, stream, few);
    if (both) {
        many.least_rows = few_rows(s) + 1;
        many.most_rows = ~0u;
        many.runs = other.runs;
        if (workspace) many.partial = workspace + bytes_of(half) / sizeof(float);
        many_grid = join_grid(s, other);
        launch_paged_flash(stream, many);
    }
    if (!few.uncut)
        hipLaunchKernelGGL((attention_paged_join<DP, 16 * G, VEC>), dim3(few_grid.x * few_grid.y + many_grid.x * many_grid.y),
                       dim3(kThreads), 0, stream, few, few_grid, many, many_grid);
    return hipGetLastError();
}

template <int DP, bool VEC>
hipError_t launch_groups(hipStream_t stream, const PagedShape &s, const PagedArgs &a, float *workspace) {
    return groups_of(s) == 2 ? launch<DP, 2, VEC>(stream, s, a, workspace) : launch<DP, 1, VEC>(stream, s, a, workspace);
}

uint32_t paged_lds_bytes(uint32_t dim, uint32_t rows) {
    const uint32_t pitch = (dim <= 64 ? 64 : 128) + 4;
    return uint32_t(kWaves * rows * (pitch * sizeof(float) + sizeof(float2)) + rows * sizeof(RowPlan) + kWaves * sizeof(uint32_t));
}

}  // namespace

LaunchShape attention_paged_shape(const PagedShape &s) {
    const Half few = few_of(s), many = many_of(s);
    // Tiles are counted in 32 bits.
    if (few.tiles > 0x7fffffffull || (has_many(s) && many.tiles > 0x7fffffffull)) return {nullptr, {0, 0, 0}, {0, 0, 0}, 0};
    if (has_many(s)) {
        static const char *const names[4] = {"attention_paged_flash_d32", "attention_paged_flash_d64",
                                             "attention_paged_flash_d96", "attention_paged_flash_d128"};
        return {names[(s.dim - 1) / 32], {many.runs, 1, 1}, {2 * many.rows, 1, 1}, paged_flash_lds_bytes(s.dim)};
    }
    static const char *const names[3][2] = {{"attention_paged_d64_r16", "attention_paged_d64_r32"},
                                            {"attention_paged_d96_r16", "attention_paged_d96_r32"},
                                            {"attention_paged_d128_r16", "attention_paged_d128_r32"}};
    return {names[s.dim <= 64 ? 0 : s.dim <= 96 ? 1 : 2][groups_of(s) - 1], {few.runs, 1, 1}, {kThreads, 1, 1}, paged_lds_bytes(s.dim, few.rows)};
}

size_t attention_paged_workspace_bytes(const PagedShape &s) {
    return uncut(s) ? 0 : bytes_of(few_of(s)) + (has_many(s) ? bytes_of(many_of(s)) : 0);
}

hipError_t attention_paged_f32(hipStream_t stream, const PagedShape &s, const PagedBuffers &x, float *workspace) {
    PagedArgs a{};
    a.q = x.q; a.k = x.k; a.v = x.v; a.tables = x.tables; a.lengths = x.lengths; a.counts = x.counts;
    a.out = x.out;
    const size_t d = s.dim;
    a.q_batch = d * s.heads * s.queries;
    a.q_head = s.token_major ? d : d * s.queries;
    a.q_row = uint32_t(s.token_major ? d * s.heads : d);
    a.p_page = d * s.kv_heads * s.page;
    a.p_head = s.pages_token_major ? d : d * s.page;
    a.p_row = uint32_t(s.pages_token_major ? d * s.kv_heads : d);
    a.batch = s.batch; a.kv_heads = s.kv_heads; a.group = s.heads / s.kv_heads; a.queries = s.queries;
    a.pages = s.pages; a.table = s.table; a.page = s.page; a.dim = s.dim;
    a.steps = s.page / 16;
    a.inverse = uint32_t(((1ull << 31) + a.steps - 1) / a.steps);
    a.qscale = (1.0f / sqrtf(float(s.dim))) * kLog2e;
    uintptr_t bits = 0;
    for (const float *y : {x.q, x.k, x.v, const_cast<const float *>(x.out)}) bits |= reinterpret_cast<uintptr_t>(y);
    if ((!workspace && !uncut(s)) || (s.dim % 4 == 0 && bits & 15u)) return hipErrorInvalidValue;  // the runtime's regions are aligned
    if (s.dim % 4)
        return s.dim <= 64 ? launch_groups<64, false>(stream, s, a, workspace) : launch_groups<128, false>(stream, s, a, workspace);
    return s.dim <= 64 ? launch_groups<64, true>(stream, s, a, workspace) : launch_groups<128, true>(stream, s, a, workspace);
}

}  // namespace hipk
}  // namespace jade
