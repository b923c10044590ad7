// Attention of a few query rows over ragged keys: a tree of drafted tokens over
// a cache (attention_tree, one node of which is ordinary decoding) and queries
// over an encoder's states (attention_cross). Every (sequence, kv head) is a
// product of its own: rows r = (head of the group, query), keys 0 .. length - 1
// and, for a tree, the drafted nodes, of which a node sees itself and its
// ancestors:
//   out_r = sum_j exp(s_rj - m_r) v_j / sum_j exp(s_rj - m_r), s_rj = q_r k_j / sqrt(dim).
// Rows without a key (a sequence of length zero, a slot without a node) are zeros.
//
// One pass with a running maximum and sum. FP32 MFMAs (16x16x4) in the
// transposed form of attention_f32.hip:
//   S^T[key, row] = sum_d K[key, d] Q[row, d],  O^T[d, row] += sum_key V^T[d, key] P^T[key, row].
// The scores leave a lane with row l % 16 of keys 4 (l / 16) + i, which is the B
// operand that the second product wants for its key step i, and both products
// contract and order dims as the 16-byte loads of K and V leave them: K, V and P
// never go through LDS, and no wave waits for another.
//
// Work is spread over the chip by tiles of 64 keys (a wave takes 16 of each): all
// tiles of all (sequence, kv head, row block)s in a row, cut into equal runs, one
// per block. A run that holds a whole (sequence, kv head, row block) writes its
// outputs; one that holds part of it leaves sums and maximum in the workspace for
// attention_ragged_join. So neither long sequences nor ragged ones leave CUs idle.
//
// This kernel takes up to 16 rows and is bound by reading K and V: 4 nodes x 32 heads (8 of
// keys) over 131072 keys of 128, 1.07 GB in 187 us, 5.7 TB/s; 16 x 24 heads of one query
// over at most 1531 keys of 80, 59 us, 4.9 TB/s; one query over 1024 keys 8.9 us, which is
// two launches and loads that wait for one another (lengths, Q, K, the partial sums). More
// rows go to the kernel on bf16 parts (attention_ragged_parts.hip): 64 nodes over 4
// sequences took 169 us with FP32 MFMAs, 64 rows a block, and take 115 to 125.
#include <cmath>

#include "attention_flash.hpp"
#include "kernels.hpp"
#include "ragged_device.hpp"

namespace jade {
namespace hipk {
namespace {

using namespace ragged;

constexpr int kTile = 64;  // keys per tile

// DP: head dim padded (64, 128).
template <int DP, bool VEC>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_ragged(RaggedArgs a) {
    constexpr int KJ = DP / 16, NJ = DP / 64, RB = 16;
    __shared__ __attribute__((aligned(16))) float part[kWaves][RB][DP + 4];
    __shared__ float2 ml[kWaves][RB];
    __shared__ RowPlan plans[RB];
    __shared__ uint64_t sees[kMaxTreeNodes][kWords];
    __shared__ int above[kMaxTreeNodes];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, g = lane >> 4;
    const uint32_t units = a.kv_heads * a.row_blocks;
    const Spread<kTile> spread(a);
    const uint32_t total = spread.total * units, chunk = (total + a.runs - 1) / a.runs;
    const uint32_t run = run_of(blockIdx.x, a.runs);
    uint32_t b, before;
    const uint32_t t_stop = spread.start(run + 1, chunk, units, b, before);
    uint32_t t = spread.start(run, chunk, units, b, before);

    const uint32_t row_bytes = a.k_row * 4u;
    uint32_t koff[KJ], voff[NJ][4];
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
        const int d = 16 * j + 4 * g;
        koff[j] = d < a.dim ? uint32_t(16 * wave + m) * row_bytes + uint32_t(d) * 4u : kDeadOffset;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 64 * j + 4 * m;
            voff[j][i] = d < a.dim ? uint32_t(16 * wave + 4 * g + i) * row_bytes + uint32_t(d) * 4u : kDeadOffset;
        }

    // The part of a (sequence, kv head, row block) that tile t of the launch begins in this
    // run; nothing where the run is over.
    struct Unit {
        uint32_t b, before, kv, rb, begin, end, tiles, len, cached;
    };
    auto unit_at = [&](uint32_t t, uint32_t b, uint32_t before) {
        Unit u{};
        if (t >= t_stop) return u;
        for (u.b = b, u.before = before;; ++u.b) {  // the run ends with a sequence that has tiles
            u.len = spread.length(u.b);
            u.cached = (u.len + kTile - 1) / kTile;
            u.tiles = u.cached + spread.draft_tiles;
            if (u.tiles) break;
        }
        const uint32_t in = t - before * units, unit = in / u.tiles;
        u.begin = in - unit * u.tiles;
        u.kv = unit / a.row_blocks;
        u.rb = unit - u.kv * a.row_blocks;
        u.end = min(u.tiles, u.begin + (t_stop - t));
        return u;
    };
    // Tile x of a unit's keys or values: its own descriptor (no offset passes 2^31, however
    // long the cache), which ends with its last key's row; past `end` it holds nothing.
    auto tile_of = [&](const float *caches, const float *drafts, const Unit &u, uint32_t x) {
        const bool drafted = x >= u.cached;
        const uint32_t at = drafted ? x - u.cached : x, left = (drafted ? a.nodes : u.len) - at * kTile;
        const size_t head = drafted ? u.b * a.d_batch + u.kv * a.d_head : u.b * a.k_batch + u.kv * a.k_head;
        const float *from = (drafted ? drafts : caches) + head + size_t(at) * kTile * a.k_row;
        const uint32_t bytes = x < u.end ? (min(left, uint32_t(kTile)) - 1) * row_bytes + uint32_t(a.dim) * 4u : 0u;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(from), 0, int(bytes), int(kRawBuffer));
    };
    // A last chunk that is not whole reads into the next row, or nothing past the tile.
    auto load = [&](__amdgpu_buffer_rsrc_t from, uint32_t at) {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, int(at), 0, 0));
    };
    f32x4 kf[KJ], vf[NJ][4], qf[KJ];
    auto load_k = [&](const Unit &u, uint32_t x) {
        const auto from = tile_of(a.k, a.kd, u, x);
#pragma unroll
        for (int j = 0; j < KJ; ++j) kf[j] = load(from, koff[j]);
    };
    auto load_v = [&](const Unit &u, uint32_t x) {
        const auto from = tile_of(a.v, a.vd, u, x);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) vf[j][i] = load(from, voff[j][i]);
    };
    uint32_t tree = ~0u;  // the sequence whose tree is in LDS
    float above_me = 0.f;
    // Q^T operand: row m of the block, dims 16 j + 4 g + e; and what the tree is made of.
    auto load_rows = [&](const Unit &u) {
        if (u.begin == u.end) return;
        if (u.end > u.cached && tree != u.b && tid < int(a.nodes)) above_me = a.parents[size_t(u.b) * a.nodes + tid];
        const uint32_t r = u.rb * RB + m, head = r / a.queries, query = r - head * a.queries;
        const float *row = a.q + u.b * a.q_batch + (size_t(u.kv) * a.group + head) * a.q_head + size_t(query) * a.q_row;
#pragma unroll
        for (int j = 0; j < KJ; ++j) qf[j] = load_dims<VEC>(head < a.group ? row : nullptr, 16 * j + 4 * g, a.dim);
    };
    Unit u = unit_at(t, b, before);
    load_k(u, u.begin);
    load_v(u, u.begin);
    load_rows(u);
    while (u.begin < u.end) {
        const uint32_t begin = u.begin, end = u.end, cached = u.cached, len = u.len;
        const bool whole = begin == 0 && end == u.tiles;
        // The unit after this one, whose first loads go beside this one's last products (64 x 32
        // heads (8 of keys) over at most 512 keys of 128, 4 nodes: 53.7 -> 51.9 us; 1024 x 4
        // heads over 64 keys of 64 72.0 -> 68.7; a launch of a tile a run 8.8 -> 8.9).
        t += end - begin;
        const bool over = t >= (u.before + u.tiles) * units;
        const Unit next = unit_at(t, u.b + over, over ? u.before + u.tiles : u.before);
        auto next_k = [&](uint32_t x) { x + 1 < end ? load_k(u, x + 1) : load_k(next, next.begin); };
        auto next_v = [&](uint32_t x) { x + 1 < end ? load_v(u, x + 1) : load_v(next, next.begin); };
#pragma unroll
        for (int j = 0; j < KJ; ++j) qf[j] *= a.qscale;  // log2 units

        f32x4 acc[NJ][4];
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 p;  // scores, then weights, of keys 16 wave + 4 g + i
        auto score = [&]() __attribute__((always_inline)) {
            if (!VEC)  // the next row's values may not be finite
#pragma unroll
                for (int j = 0; j < KJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (16 * j + 4 * g + e >= a.dim) kf[j][e] = 0.f;
            p = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) p = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][e], qf[j][e], p, 0, 0, 0);
        };
        auto weigh = [&]() __attribute__((always_inline)) {
            const float most = fmaxf(fmaxf(p.x, p.y), fmaxf(p.z, p.w));
            if (__any(most > top + kLazyMax)) {
                const float reached = fmaxf(top, across_keys_max(most));
                const float keep = reached == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - reached);
                top = reached;
                sum *= keep;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][e] *= keep;
            }
            const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = __builtin_amdgcn_exp2f(p[i] - from);
                sum += p[i];
            }
        };
        auto add = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[j][i][e], p[i], acc[j][e], 0, 0, 0);
        };
        uint32_t x = begin;
        for (; x < min(end, cached); ++x) {
            score();
            next_k(x);
            if ((x + 1) * kTile > len) {
                const int first = int(x) * kTile + 16 * wave + 4 * g;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (first + i >= int(len)) p[i] = -INFINITY;
            }
            weigh();
            add();
            next_v(x);
        }

        if (end > cached) {
            if (tree != u.b) see_ancestors(a.nodes, above_me, sees, above);
            tree = u.b;
            const uint32_t query = (u.rb * RB + m) % a.queries;  // queries == nodes; rows past the last see as others do
            for (; x < end; ++x) {
                score();
                next_k(x);
                const uint64_t seen = sees[query][x - cached];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!(seen >> (16 * wave + 4 * g + i) & 1)) p[i] = -INFINITY;
                weigh();
                bool odd = false;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) odd |= !finite(vf[j][i][e]);
                if (!__any(odd)) {
                    add();
                } else {
                    // A drafted value that is not finite, which not every row may see: the
                    // finite ones, then the weight that each row gives to each special one.
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int k = -1; k < 3; ++k) {
                                __builtin_amdgcn_sched_barrier(0);  // one at a time: a rare path takes no registers
                                f32x4 sums = k < 0 ? acc[j][e] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float v = vf[j][i][e], u = k >= 0 ? is(k, v) : finite(v) ? v : 0.f;
                                    sums = __builtin_amdgcn_mfma_f32_16x16x4f32(u, p[i], sums, 0, 0, 0);
                                }
                                if (k < 0)
                                    acc[j][e] = sums;
                                else
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        if (sums[i] > 0.f) acc[j][e][i] += special(k);
                            }
                }
                next_v(x);
            }
        }
        load_rows(next);

        // The four waves' sums joined: row m, dims 64 j + 16 g + 4 i + e.
        __syncthreads();
        const float all = across_keys_sum(sum);
        if (g == 0) ml[wave][m] = float2{top, all};
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4 *>(&part[wave][m][64 * j + 16 * g + 4 * i]) =
                    f32x4{acc[j][0][i], acc[j][1][i], acc[j][2][i], acc[j][3][i]};
        __syncthreads();
        finish<DP, RB, VEC>(a, run, u.b, u.kv, u.rb, whole, begin == 0, part, ml, plans, sees, 1.f);
        u = next;
    }
}

// What the runs left of a (sequence, kv head, row block) cut between them, and the
// zeros of sequences without keys. Blocks x go over the units: unit x itself where there
// are at most `runs` units, else the one that the cut before run x is the first of. DP / 4
// lanes have a row; ROWS rows of a unit go to a block, each with all of its slots, or
// (ROWS 1) one, with the slots shared out (a unit of many runs).
template <int DP, int RB, int TILE, int ROWS, bool VEC>
__global__ __launch_bounds__(kThreads) void attention_ragged_join(RaggedArgs a) {
    constexpr int LANES = DP / 4, PARTS = kThreads / LANES / ROWS;
    __shared__ __attribute__((aligned(16))) f32x4 sums[PARTS][LANES];
    __shared__ float2 weights[PARTS];
    const int tid = threadIdx.x, lane = tid % LANES, p = ROWS == 1 ? tid / LANES : 0;
    const uint32_t units = a.kv_heads * a.row_blocks, row = blockIdx.y * ROWS + (ROWS == 1 ? 0 : tid / LANES), d = 4 * lane;
    const bool by_unit = a.batch * units <= a.runs;
    const Spread<TILE> spread(a);
    const uint32_t chunk = (spread.total * units + a.runs - 1) / a.runs;
    uint32_t b, unit, start, tiles;
    if (by_unit) {
        b = blockIdx.x / units;
        unit = blockIdx.x - b * units;
        tiles = spread.tiles_at(b);
        start = spread.before(b) * units + unit * tiles;
    } else {
        if (!spread.draft_tiles)
            for (b = blockIdx.x; b < a.batch; b += a.runs) {
                if (spread.tiles_at(b)) continue;
                const size_t n = size_t(a.kv_heads) * a.group * a.queries * a.dim;
                float *out = a.out + size_t(b) * a.q_batch;
                for (size_t i = blockIdx.y * kThreads + tid; i < n; i += gridDim.y * kThreads) out[i] = 0.f;
            }
        uint32_t before;
        const uint32_t cut = spread.start(blockIdx.x, chunk, units, b, before);
        if (cut == 0 || cut == spread.total * units) return;
        tiles = spread.tiles_at(b);
        if (!tiles) return;  // at a sequence's start
        unit = (cut - before * units) / tiles;
        start = before * units + unit * tiles;
        if (start + chunk < cut || start == cut) return;  // not its first cut
    }
    const uint32_t kv = unit / a.row_blocks, rb = unit - kv * a.row_blocks;
    const bool mine = row < min(uint32_t(RB), a.group * a.queries - rb * RB);
    if (!tiles) {
        if (p == 0 && mine) store_row<VEC>(a, b, kv, rb * RB + row, d, f32x4{0.f, 0.f, 0.f, 0.f}, 1.f);
        return;
    }
    const uint32_t first = start / chunk, last = (start + tiles - 1) / chunk;
    if (first == last || spread.rounds(tiles, chunk)) return;
    const float2 *ml = reinterpret_cast<const float2 *>(a.partial + 2 * size_t(a.runs) * RB * DP);
    // A unit's first run had it last, the others first.
    auto slot = [&](uint32_t r) { return (2 * size_t(r) + (r == first)) * RB + row; };
    float most = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    auto join = [&](float top, float sum, f32x4 outs) {
        const float next = fmaxf(most, top), from = next == -INFINITY ? 0.f : next;
        const float old = __builtin_amdgcn_exp2f(most - from), weight = __builtin_amdgcn_exp2f(top - from);
        most = next;
        l = l * old + sum * weight;
        o = o * old + outs * weight;
    };
    if (mine) {
#pragma unroll 4
        for (uint32_t r = first + p; r <= last; r += PARTS) {
            const float2 x = ml[slot(r)];
            join(x.x, x.y, *reinterpret_cast<const f32x4 *>(a.partial + slot(r) * DP + d));
        }
    }
    if constexpr (PARTS > 1) {
        sums[p][lane] = o;
        if (lane == 0) weights[p] = float2{most, l};
        __syncthreads();
        if (p) return;
#pragma unroll
        for (int x = 1; x < PARTS; ++x) join(weights[x].x, weights[x].y, sums[x][lane]);
    }
    if (mine) store_row<VEC>(a, b, kv, rb * RB + row, d, o, l);
}

uint32_t rows_of(const RaggedShape &s) { return s.heads / s.kv_heads * s.queries; }

// More than 16 rows go to the kernel on bf16 parts, where a tile of its 128 keys spans less
// than 2 GiB.
bool on_parts(const RaggedShape &s) {
    return rows_of(s) > 16 && (!s.token_major || uint64_t(s.kv_heads) * s.dim < 1u << 22);
}
uint32_t block_rows(const RaggedShape &s) { return !on_parts(s) ? 16 : rows_of(s) <= 32 ? 32 : 64; }
uint32_t row_blocks(const RaggedShape &s) { return (rows_of(s) + block_rows(s) - 1) / block_rows(s); }

// Tiles of a (sequence, kv head, row block) of full length, and of a launch of such.
uint32_t unit_tiles(const RaggedShape &s) {
    const uint32_t tile = on_parts(s) ? kPartsTile : kTile;
    return (s.keys + tile - 1) / tile + (s.nodes + tile - 1) / tile;
}
uint64_t ragged_tiles(const RaggedShape &s) { return uint64_t(s.batch) * s.kv_heads * row_blocks(s) * unit_tiles(s); }

// Queries of an encoder's states may go to the flash kernel (attention_flash.hip), which
// splits K and V once for 128 or 256 rows but has one block for them and all their keys.
// Both are estimated, in us, from what they measured: the flash kernel 8 and, for every 256
// blocks, 1.7 (dims to 64), 3.6 (to 96) or 4.6 for 32 keys of full blocks, 0.35 of that for
// empty ones; the kernel on parts 2.8, 4.1 or 5.9 for 128 keys, 8, 9.5 or 11 for each unit a
// run begins, and 3 for the join. Measured, flash and parts: 4 x 32 heads (8 of keys) x 1000
// queries x 4096 keys of 128 1179 and 1385 us; 32 x 16 x 200 x 100 of 128 48 and 129; 32 x
// 16 x 80 x 128 of 64 21 and 43; 16 x 3000 x 1500 of 128 198 and 220; 4 x 32 x 256 x 2048
// of 128 256 and 221, of 96 212 and 170; 16 x 1500 x 1500 of 64 82 and 71, of 80 154 and 93;
// 16 x 3000 x 1500 of 96 160 and 178; 4 x 8 x 256 x 1024 of 128 131 and 40.
bool on_flash(const RaggedShape &s) {
    const uint64_t d = s.dim, heads = uint64_t(s.batch) * s.kv_heads, rows = rows_of(s), fb = flash_ragged_rows(s.dim);
    const uint64_t q_span = s.token_major ? d * s.heads * s.queries : d * rows;
    const uint64_t k_span = (s.token_major ? d * s.kv_heads : d) * (s.keys + 128ull);
    // Offsets of a head's rows in 31 bits, tiles past the last one in 32; grid.y, and the
    // threads along grid.x (2 fb a block).
    if (!on_parts(s) || s.dim % 4 || s.nodes || q_span >= 1u << 29 || k_span >= 1u << 29) return false;
    if ((rows + fb - 1) / fb > 65535 || heads * 2 * fb > 0xffffffffull) return false;
    const uint64_t blocks = heads * ((rows + fb - 1) / fb), units = heads * row_blocks(s);
    const double full = double(rows) / double((rows + fb - 1) / fb * fb);
    const double flash = 8.0 + double((blocks + kCus - 1) / kCus) * double((s.keys + 31) / 32) *
                                   (d <= 64 ? 1.7 : d <= 96 ? 3.6 : 4.6) * (0.35 + 0.65 * full);
    const double parts = 3.0 + double((ragged_tiles(s) + kCus - 1) / kCus) * (d <= 64 ? 2.8 : d <= 96 ? 4.1 : 5.9) +
                         double((units + kCus - 1) / kCus) * (d <= 64 ? 8.0 : d <= 96 ? 9.5 : 11.0);
    return flash < parts;
}

// Runs of a launch: as many blocks as work best on a CU, or one per tile where there can be
// no more tiles.
// 16 rows: two. Three, where the registers allow it (dims to 64): 36 x 20 heads x 1101 keys
// 61.6 -> 57.0 us, but 8 x 16 x 4096 52.4 -> 55.1 and 64 x 8 x 100 11.3 -> 13.3.
// On parts one, which overlaps its own work; but two of 32 rows and dims to 64, which the
// registers allow, where units are short and mostly begin and end: 19 nodes x 50 x 16 heads
// over 119 keys of 40 42.0 -> 32.4, 28 nodes x 5 x 28 heads over at most 1391 of 18 35.0 ->
// 24.7, but 30 nodes x 2 x 8 heads over at most 5000 of 33 24.4 -> 26.4.
uint32_t runs_of(const RaggedShape &s) {
    const uint64_t tiles = ragged_tiles(s);
    const bool two = !on_parts(s) || (block_rows(s) == 32 && s.dim <= 64 && unit_tiles(s) <= 16);
    const uint32_t most = two ? 2 * kCus : kCus;
    return tiles >= most ? most : uint32_t((tiles + 7) / 8 * 8);
}

template <int DP, int RB, int TILE, bool VEC>
void launch_join(hipStream_t stream, const RaggedArgs &a) {
    constexpr uint32_t kRowsOf = kThreads / (DP / 4);  // rows of a block
    const uint32_t units = a.batch * a.kv_heads * a.row_blocks, all = a.group * a.queries, rows = all < RB ? all : RB;
    const uint32_t x = units < a.runs ? units : a.runs;
    // Units of 16 runs or more: their slots are shared out (with the attention itself, 4 nodes over 131072
    // keys, 64 runs a unit: 186 us so, 193 by whole rows); else whole rows (64 nodes x 4 heads
    // over 4 sequences of 4096 keys: 133 us shared, 122 by rows).
    if (16 * units <= a.runs)
        hipLaunchKernelGGL((attention_ragged_join<DP, RB, TILE, 1, VEC>), dim3(x, rows), dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((attention_ragged_join<DP, RB, TILE, kRowsOf, VEC>), dim3(x, (rows + kRowsOf - 1) / kRowsOf),
                           dim3(kThreads), 0, stream, a);
}

template <int DP, bool VEC>
hipError_t launch_rows(hipStream_t stream, const RaggedArgs &a, uint32_t rb) {
    if (rb == 16) {
        hipLaunchKernelGGL((attention_ragged<DP, VEC>), dim3(a.runs), dim3(kThreads), 0, stream, a);
        launch_join<DP, 16, kTile, VEC>(stream, a);
    } else {
        launch_ragged_parts(stream, a, rb);
        rb == 32 ? launch_join<DP, 32, kPartsTile, VEC>(stream, a) : launch_join<DP, 64, kPartsTile, VEC>(stream, a);
    }
    return hipGetLastError();
}

uint32_t ragged_lds_bytes(uint32_t dim, uint32_t rb) {
    if (rb > 16) return ragged_parts_lds_bytes(dim, rb);
    const uint32_t pitch = (dim <= 64 ? 64 : 128) + 4;
    return uint32_t(kWaves * rb * (pitch * sizeof(float) + sizeof(float2)) + rb * sizeof(RowPlan) +
                    kMaxTreeNodes * (kWords * sizeof(uint64_t) + sizeof(int)));
}

}  // namespace

LaunchShape attention_ragged_shape(const RaggedShape &s) {
    if (on_flash(s)) {
        static const char *const names[4] = {"attention_flash_ragged_d32", "attention_flash_ragged_d64",
                                             "attention_flash_ragged_d96", "attention_flash_ragged_d128"};
        const uint32_t rb = flash_ragged_rows(s.dim);
        return {names[(s.dim - 1) / 32], {s.batch * s.kv_heads, (rows_of(s) + rb - 1) / rb, 1}, {2 * rb, 1, 1},
                attention_flash_lds_bytes(s.dim, int(rb / 32))};
    }
    // Tiles are counted in 32 bits.
    if (ragged_tiles(s) > 0x7fffffffull) return {nullptr, {0, 0, 0}, {0, 0, 0}, 0};
    const uint32_t rb = block_rows(s), wide = s.dim <= 64 ? 0 : s.dim <= 96 ? 1 : 2;
    static const char *const names[3][3] = {
        {"attention_ragged_d64", "attention_ragged_parts_d64_r32", "attention_ragged_parts_d64_r64"},
        {"attention_ragged_d128", "attention_ragged_parts_d96_r32", "attention_ragged_parts_d96_r64"},
        {"attention_ragged_d128", "attention_ragged_parts_d128_r32", "attention_ragged_parts_d128_r64"}};
    return {names[wide][rb / 32], {runs_of(s), 1, 1}, {kThreads, 1, 1}, ragged_lds_bytes(s.dim, rb)};
}

size_t attention_ragged_workspace_bytes(const RaggedShape &s) {
    if (on_flash(s)) return 0;
    const size_t rb = block_rows(s), dp = s.dim > 64 ? 128 : 64;
    return 2 * size_t(runs_of(s)) * rb * (dp + 2) * sizeof(float);
}

hipError_t attention_ragged_f32(hipStream_t stream, const RaggedShape &s, const RaggedBuffers &x, float *workspace) {
    RaggedArgs a{};
    a.q = x.q; a.k = x.k; a.v = x.v; a.lengths = x.lengths; a.kd = x.k_draft; a.vd = x.v_draft; a.parents = x.parents;
    a.out = x.out;
    a.partial = workspace;
    const size_t d = s.dim;
    a.q_batch = d * s.heads * s.queries;
    a.k_batch = d * s.kv_heads * s.keys;
    a.d_batch = d * s.kv_heads * s.nodes;
    a.q_head = s.token_major ? d : d * s.queries;
    a.k_head = s.token_major ? d : d * s.keys;
    a.d_head = s.token_major ? d : d * s.nodes;
    a.q_row = uint32_t(s.token_major ? d * s.heads : d);
    a.k_row = uint32_t(s.token_major ? d * s.kv_heads : d);
    a.batch = s.batch; a.kv_heads = s.kv_heads; a.group = s.heads / s.kv_heads; a.queries = s.queries;
    a.keys = s.keys; a.nodes = s.nodes; a.dim = s.dim;
    a.row_blocks = row_blocks(s);
    a.runs = runs_of(s);
    a.qscale = (1.0f / sqrtf(float(s.dim))) * kLog2e;
    uintptr_t bits = 0;
    for (const float *y : {x.q, x.k, x.v, x.k_draft, x.v_draft, const_cast<const float *>(x.out)})
        bits |= reinterpret_cast<uintptr_t>(y);
    if (s.dim % 4 == 0 && bits & 15u) return hipErrorInvalidValue;  // the runtime's regions are aligned
    if (on_flash(s)) return launch_flash_ragged(stream, a);
    if (!workspace) return hipErrorInvalidValue;
    const uint32_t rb = block_rows(s);
    if (s.dim % 4) return s.dim <= 64 ? launch_rows<64, false>(stream, a, rb) : launch_rows<128, false>(stream, a, rb);
    return s.dim <= 64 ? launch_rows<64, true>(stream, a, rb) : launch_rows<128, true>(stream, a, rb);
}

}  // namespace hipk
}  // namespace jade
