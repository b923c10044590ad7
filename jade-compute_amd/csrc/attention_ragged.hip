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
#include <cmath>

#include "attention_ragged.hpp"
#include "kernels.hpp"
#include "whole.hpp"

namespace jade {
namespace hipk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kTile = 64;   // keys per tile
constexpr uint32_t kWorkers = 512;  // runs: two blocks per CU
constexpr float kLazyMax = 8.0f;   // log2 units: the running maximum moves only past this
constexpr uint32_t kRawBuffer = 0x00020000;    // buffer descriptor word 3: raw buffer, 32-bit data format
constexpr uint32_t kDeadOffset = 0x80000000u;  // past every tile: reads zero
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kWords = int(kMaxTreeNodes) / 64;

// Tiles of one (kv head, row block) of sequence b.
__device__ inline uint32_t tiles_of(const RaggedArgs &a, uint32_t b, uint32_t draft_tiles) {
    return (whole_below(a.lengths[b], a.keys) + kTile - 1) / kTile + draft_tiles;
}
__device__ inline uint32_t scan_add(uint32_t x, int lane) {
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const uint32_t y = __shfl_up(x, step);
        if (lane >= step) x += y;
    }
    return x;
}
__device__ inline uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// Tiles of all sequences (of one (kv head, row block) each).
__device__ inline uint32_t all_tiles(const RaggedArgs &a, uint32_t draft_tiles) {
    const int lane = threadIdx.x & 63;
    uint32_t sum = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
        const uint32_t b = b0 + lane;
        sum += uniform(__shfl(scan_add(b < a.batch ? tiles_of(a, b, draft_tiles) : 0, lane), 63));
    }
    return sum;
}
// The sequence with tile `t` < all_tiles() and the tiles before it.
__device__ inline void find_sequence(const RaggedArgs &a, uint32_t draft_tiles, uint32_t t, uint32_t &b,
                                     uint32_t &before) {
    const int lane = threadIdx.x & 63;
    before = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
        const uint32_t at = b0 + lane;
        const uint32_t own = at < a.batch ? tiles_of(a, at, draft_tiles) : 0, up_to = scan_add(own, lane);
        const uint64_t past = __ballot(before + up_to > t);
        if (past) {
            const int first = __builtin_ctzll(past);
            b = b0 + first;
            before = uniform(before + __shfl(up_to - own, first));
            return;
        }
        before += uniform(__shfl(up_to, 63));
    }
    b = a.batch;  // not reached
}

__device__ inline bool is_node(float parent, int n) {
    return parent == -1.f || (parent >= 0.f && parent < float(n) && parent == truncf(parent));
}

// Run w of the launch: runs of one XCD are neighbours, so the row blocks of one kv
// head, which read the same keys, meet in its L2.
__device__ inline uint32_t run_of(uint32_t id, uint32_t runs) { return id % 8 * (runs / 8) + id / 8; }

__device__ inline float across_keys_max(float x) { return fmaxf(fmaxf(x, __shfl_xor(x, 16)), fmaxf(__shfl_xor(x, 32), __shfl_xor(x, 48))); }
__device__ inline float across_keys_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// Row r of (sequence b, kv head): its sums o of dims d .. d + 3 over its weights' sum.
template <bool VEC>
__device__ inline void store_row(const RaggedArgs &a, uint32_t b, uint32_t kv, uint32_t r, uint32_t d, f32x4 o, float l) {
    const uint32_t head = r / a.queries, query = r - head * a.queries;
    const bool node = !a.nodes || is_node(a.parents[size_t(b) * a.nodes + query], int(query));
    o = node ? o * (1.0f / l) : f32x4{0.f, 0.f, 0.f, 0.f};
    float *out = a.out + size_t(b) * a.q_batch + (size_t(kv) * a.group + head) * a.q_head + size_t(query) * a.q_row;
    if (VEC) {
        if (d < a.dim) *reinterpret_cast<f32x4 *>(out + d) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < a.dim) out[d + e] = o[e];
    }
}

// DP: head dim padded (64, 128); QT: row tiles of 16 per block; VEC: rows of whole
// float4s, 16-byte aligned.
template <int DP, int QT, bool VEC>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_ragged(RaggedArgs a) {
    constexpr int KJ = DP / 16, NJ = DP / 64, RB = 16 * QT, PITCH = DP + 4;
    __shared__ __attribute__((aligned(16))) float part[kWaves][RB][PITCH];
    __shared__ float2 ml[kWaves][RB];
    __shared__ uint64_t sees[kMaxTreeNodes][kWords];
    __shared__ int above[kMaxTreeNodes];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, g = lane >> 4;
    const uint32_t draft_tiles = (a.nodes + kTile - 1) / kTile, units = a.kv_heads * a.row_blocks;
    const uint32_t total = all_tiles(a, draft_tiles) * units, chunk = (total + a.runs - 1) / a.runs;
    const uint32_t run = run_of(blockIdx.x, a.runs);
    if (uint64_t(run) * chunk >= total) return;
    uint32_t t = run * chunk;
    const uint32_t t_stop = min(total, t + chunk);
    uint32_t b, before;
    find_sequence(a, draft_tiles, t / units, b, before);

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

    while (t < t_stop) {
        const uint32_t len = uniform(whole_below(a.lengths[b], a.keys));
        const uint32_t cached = (len + kTile - 1) / kTile, tiles = cached + draft_tiles;
        if (!tiles) {
            ++b;
            continue;
        }
        const uint32_t in = t - before * units, unit = in / tiles, begin = in - unit * tiles;
        const uint32_t kv = unit / a.row_blocks, rb = unit - kv * a.row_blocks;
        const uint32_t end = min(tiles, begin + (t_stop - t));
        const bool whole = begin == 0 && end == tiles;

        if (end > cached) {  // the tree: bit n' of row n where node n sees node n'
            __syncthreads();
            const int n = tid;
            int parent = -2;
            if (n < int(a.nodes)) {
                const float p = a.parents[size_t(b) * a.nodes + n];
                parent = is_node(p, n) ? int(p) : -2;
                above[n] = parent;
#pragma unroll
                for (int w = 0; w < kWords; ++w) sees[n][w] = parent != -2 && n / 64 == w ? 1ull << (n & 63) : 0ull;
            }
            // Ancestors by doubling: after k steps a node has those up to 2^k above it.
            for (uint32_t reach = 1; reach < a.nodes; reach *= 2) {
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

        // Q^T operand, in log2 units: row m of tile qt, dims 16 j + 4 g + e.
        f32x4 qf[QT][KJ];
        int node[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            const uint32_t r = rb * RB + 16 * qt + m, head = r / a.queries, query = r - head * a.queries;
            node[qt] = int(query);
            const bool live = head < a.group;
            const float *row = a.q + size_t(b) * a.q_batch + (size_t(kv) * a.group + head) * a.q_head + size_t(query) * a.q_row;
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                const int d = 16 * j + 4 * g;
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
                if (VEC) {
                    if (live && d < a.dim) x = *reinterpret_cast<const f32x4 *>(row + d);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (live && d + e < a.dim) x[e] = row[d + e];
                }
                qf[qt][j] = x * a.qscale;
            }
        }

        const float *kb = a.k + size_t(b) * a.k_batch + size_t(kv) * a.k_head;
        const float *vb = a.v + size_t(b) * a.k_batch + size_t(kv) * a.k_head;
        const float *kd = a.kd + size_t(b) * a.d_batch + size_t(kv) * a.d_head;
        const float *vd = a.vd + size_t(b) * a.d_batch + size_t(kv) * a.d_head;
        // Tile x of a tensor: its own descriptor (no offset passes 2^31, however long
        // the cache), which ends with its last key's row; past `end` it holds nothing.
        auto tile_of = [&](const float *cache, const float *draft, uint32_t x) {
            const bool drafted = x >= cached;
            const uint32_t at = drafted ? x - cached : x, left = (drafted ? a.nodes : len) - at * kTile;
            const float *from = (drafted ? draft : cache) + size_t(at) * kTile * a.k_row;
            const uint32_t bytes = x < end ? (min(left, uint32_t(kTile)) - 1) * row_bytes + uint32_t(a.dim) * 4u : 0u;
            return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(from), 0, int(bytes), int(kRawBuffer));
        };
        auto load = [&](__amdgpu_buffer_rsrc_t from, uint32_t at, int d) {
            if (VEC) return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, int(at), 0, 0));
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = __builtin_bit_cast(
                    float, __builtin_amdgcn_raw_buffer_load_b32(from, int(d + e < a.dim ? at + 4u * e : kDeadOffset), 0, 0));
            return x;
        };
        f32x4 kf[KJ], vf[NJ][4];
        auto load_k = [&](uint32_t x) {
            const auto from = tile_of(kb, kd, x);
#pragma unroll
            for (int j = 0; j < KJ; ++j) kf[j] = load(from, koff[j], 16 * j + 4 * g);
        };
        auto load_v = [&](uint32_t x) {
            const auto from = tile_of(vb, vd, x);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) vf[j][i] = load(from, voff[j][i], 64 * j + 4 * m);
        };

        f32x4 acc[QT][NJ][4];
        float top[QT], sum[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            top[qt] = -INFINITY;
            sum[qt] = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[qt][j][e] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        load_k(begin);
        load_v(begin);
        for (uint32_t x = begin; x < end; ++x) {
            f32x4 p[QT];
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) p[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt)
                        p[qt] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][e], qf[qt][j][e], p[qt], 0, 0, 0);
            load_k(x + 1);
            const bool drafted = x >= cached;
            const int first = int(drafted ? x - cached : x) * kTile + 16 * wave + 4 * g;  // this lane's key i = 0
            if (drafted) {
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) {
                    const uint64_t word = node[qt] < int(a.nodes) ? sees[node[qt]][x - cached] : 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(word >> ((first + i) & 63) & 1)) p[qt][i] = -INFINITY;
                }
            } else if ((x + 1) * kTile > len) {
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (first + i >= int(len)) p[qt][i] = -INFINITY;
            }
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                const float most = fmaxf(fmaxf(p[qt].x, p[qt].y), fmaxf(p[qt].z, p[qt].w));
                if (__any(most > top[qt] + kLazyMax)) {
                    const float reached = fmaxf(top[qt], across_keys_max(most));
                    const float keep = reached == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top[qt] - reached);
                    top[qt] = reached;
                    sum[qt] *= keep;
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[qt][j][e] *= keep;
                }
                const float from = top[qt] == -INFINITY ? 0.f : top[qt];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[qt][i] = __builtin_amdgcn_exp2f(p[qt][i] - from);
                    sum[qt] += p[qt][i];
                }
            }
            bool odd = false;  // a drafted value that is not finite: not every row may see it
            if (drafted) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!(fabsf(vf[j][i][e]) < INFINITY)) {
                                vf[j][i][e] = 0.f;
                                odd = true;
                            }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int qt = 0; qt < QT; ++qt)
                            acc[qt][j][e] =
                                __builtin_amdgcn_mfma_f32_16x16x4f32(vf[j][i][e], p[qt][i], acc[qt][j][e], 0, 0, 0);
            load_v(x + 1);
            if (drafted && __any(odd)) {
                for (int key = 0; key < 16; ++key) {
                    const int at = int(x - cached) * kTile + 16 * wave + key;
                    if (at >= int(a.nodes)) break;
                    const float *row = vd + size_t(at) * a.k_row;
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt) {
                        const float weight = __shfl(key & 2 ? (key & 1 ? p[qt].w : p[qt].z) : (key & 1 ? p[qt].y : p[qt].x),
                                                    16 * (key >> 2) + m);
                        if (node[qt] >= int(a.nodes) || !(sees[node[qt]][at / 64] >> (at & 63) & 1)) continue;
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int d = 64 * j + 16 * g + 4 * i + e;
                                    const float v = d < a.dim ? row[d] : 0.f;
                                    if (!(fabsf(v) < INFINITY)) acc[qt][j][e][i] += weight * v;
                                }
                    }
                }
            }
        }

        // The four waves' sums joined.
        __syncthreads();
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            const float all = across_keys_sum(sum[qt]);
            if (g == 0) ml[wave][16 * qt + m] = float2{top[qt], all};
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4 *>(&part[wave][16 * qt + m][64 * j + 16 * g + 4 * i]) =
                        f32x4{acc[qt][j][0][i], acc[qt][j][1][i], acc[qt][j][2][i], acc[qt][j][3][i]};
        }
        __syncthreads();
        const uint32_t rows = min(uint32_t(RB), a.group * a.queries - rb * RB);
        const size_t slot = 2 * size_t(run) + (begin == 0);
        for (uint32_t at = tid; at < rows * (DP / 4); at += kThreads) {
            const uint32_t row = at / (DP / 4), d = at % (DP / 4) * 4;
            float most = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) most = fmaxf(most, ml[w][row].x);
            const float from = most == -INFINITY ? 0.f : most;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float weight = __builtin_amdgcn_exp2f(ml[w][row].x - from);
                l = fmaf(weight, ml[w][row].y, l);
                o += weight * *reinterpret_cast<const f32x4 *>(&part[w][row][d]);
            }
            if (whole) {
                store_row<VEC>(a, b, kv, rb * RB + row, d, o, l);
            } else {
                *reinterpret_cast<f32x4 *>(a.partial + (slot * RB + row) * DP + d) = o;
                if (d == 0)
                    reinterpret_cast<float2 *>(a.partial + 2 * size_t(a.runs) * RB * DP)[slot * RB + row] = float2{most, l};
            }
        }
        t += end - begin;
        if (t >= (before + tiles) * units) {
            before += tiles;
            ++b;
        }
    }
}

// What the runs left of a (sequence, kv head, row block) cut between them. Block x
// looks at the cut before run x and joins the unit if that is its first one; block y
// takes two rows of it. Sequences without keys get their zeros here.
template <int DP, int QT, bool VEC>
__global__ __launch_bounds__(kThreads) void attention_ragged_join(RaggedArgs a) {
    constexpr int RB = 16 * QT, LANES = DP / 4, PARTS = kThreads / (2 * LANES);
    __shared__ __attribute__((aligned(16))) f32x4 sums[PARTS][2 * LANES];
    __shared__ float weights[PARTS][2 * LANES];
    const uint32_t draft_tiles = (a.nodes + kTile - 1) / kTile, units = a.kv_heads * a.row_blocks;
    if (!draft_tiles)
        for (uint32_t b = blockIdx.x; b < a.batch; b += a.runs) {
            if (whole_below(a.lengths[b], a.keys)) continue;
            const size_t n = size_t(a.kv_heads) * a.group * a.queries * a.dim;
            float *out = a.out + size_t(b) * a.q_batch;
            for (size_t i = blockIdx.y * kThreads + threadIdx.x; i < n; i += gridDim.y * kThreads) out[i] = 0.f;
        }
    const uint32_t total = all_tiles(a, draft_tiles) * units, chunk = (total + a.runs - 1) / a.runs;
    const uint32_t run = blockIdx.x;
    if (run == 0 || uint64_t(run) * chunk >= total) return;
    const uint32_t t = run * chunk;
    uint32_t b, before;
    find_sequence(a, draft_tiles, t / units, b, before);
    const uint32_t tiles = uniform(tiles_of(a, b, draft_tiles)), in = t - before * units, unit = in / tiles;
    const uint32_t begin = in - unit * tiles, kv = unit / a.row_blocks, rb = unit - kv * a.row_blocks;
    if (begin == 0 || begin > chunk) return;
    const uint32_t first = run - 1, last = (t - begin + tiles - 1) / chunk;
    const uint32_t rows = min(uint32_t(RB), a.group * a.queries - rb * RB);
    if (2 * blockIdx.y >= rows) return;
    const int tid = threadIdx.x, at = tid % (2 * LANES), p = tid / (2 * LANES);
    const uint32_t row = 2 * blockIdx.y + at / LANES, d = at % LANES * 4;
    const float2 *ml = reinterpret_cast<const float2 *>(a.partial + 2 * size_t(a.runs) * RB * DP);
    // A unit's first run had it last, the others first.
    auto slot = [&](uint32_t r) { return (2 * size_t(r) + (r == first)) * RB + row; };
    float most = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (row < rows) {
        for (uint32_t r = first; r <= last; ++r) most = fmaxf(most, ml[slot(r)].x);
        const float from = most == -INFINITY ? 0.f : most;
        for (uint32_t r = first + p; r <= last; r += PARTS) {
            const float2 x = ml[slot(r)];
            const float weight = __builtin_amdgcn_exp2f(x.x - from);
            l = fmaf(weight, x.y, l);
            o += weight * *reinterpret_cast<const f32x4 *>(a.partial + slot(r) * DP + d);
        }
    }
    sums[p][at] = o;
    weights[p][at] = l;
    __syncthreads();
    if (p || row >= rows) return;
#pragma unroll
    for (int x = 1; x < PARTS; ++x) {
        o += sums[x][at];
        l += weights[x][at];
    }
    store_row<VEC>(a, b, kv, rb * RB + row, d, o, l);
}

struct Plan {
    uint32_t row_blocks;
    bool two;  // two row tiles of 16 per block
};
Plan plan_of(uint32_t rows) { return {rows <= 16 ? 1u : (rows + 31) / 32, rows > 16}; }

template <int DP, int QT>
hipError_t launch(hipStream_t stream, const RaggedArgs &a, bool vec) {
    const dim3 grid(a.runs), join(a.runs, 8 * QT), block(kThreads);
    if (vec) {
        hipLaunchKernelGGL((attention_ragged<DP, QT, true>), grid, block, 0, stream, a);
        hipLaunchKernelGGL((attention_ragged_join<DP, QT, true>), join, block, 0, stream, a);
    } else {
        hipLaunchKernelGGL((attention_ragged<DP, QT, false>), grid, block, 0, stream, a);
        hipLaunchKernelGGL((attention_ragged_join<DP, QT, false>), join, block, 0, stream, a);
    }
    return hipGetLastError();
}

uint64_t ragged_tiles(const RaggedShape &s) {
    const uint64_t tiles = (uint64_t(s.keys) + kTile - 1) / kTile + (s.nodes + kTile - 1) / kTile;
    return uint64_t(s.batch) * s.kv_heads * plan_of(s.heads / s.kv_heads * s.queries).row_blocks * tiles;
}

// Runs of a launch: kWorkers, or one per tile where there can be no more tiles.
uint32_t runs_of(const RaggedShape &s) {
    const uint64_t tiles = ragged_tiles(s);
    return tiles >= kWorkers ? kWorkers : uint32_t((tiles + 7) / 8 * 8);
}

}  // namespace

LaunchShape attention_ragged_shape(const RaggedShape &s) {
    // Tiles are counted in 32 bits.
    if (ragged_tiles(s) > 0x7fffffffull) return {nullptr, {0, 0, 0}, {0, 0, 0}, 0};
    const bool two = plan_of(s.heads / s.kv_heads * s.queries).two, wide = s.dim > 64;
    static const char *const names[2][2] = {{"attention_ragged_d64_r16", "attention_ragged_d64_r32"},
                                            {"attention_ragged_d128_r16", "attention_ragged_d128_r32"}};
    const uint32_t rb = two ? 32 : 16, pitch = (wide ? 128 : 64) + 4;
    return {names[wide][two], {runs_of(s), 1, 1}, {kThreads, 1, 1},
            uint32_t(kWaves * rb * (pitch * sizeof(float) + sizeof(float2)) +
                     kMaxTreeNodes * (kWords * sizeof(uint64_t) + sizeof(int)))};
}

size_t attention_ragged_workspace_bytes(const RaggedShape &s) {
    const size_t rb = plan_of(s.heads / s.kv_heads * s.queries).two ? 32 : 16, dp = s.dim > 64 ? 128 : 64;
    return 2 * size_t(runs_of(s)) * rb * (dp + 2) * sizeof(float);
}

hipError_t attention_ragged_f32(hipStream_t stream, const RaggedShape &s, const RaggedBuffers &x, float *workspace) {
    if (!workspace) return hipErrorInvalidValue;
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
    const Plan p = plan_of(a.group * s.queries);
    a.row_blocks = p.row_blocks;
    a.runs = runs_of(s);
    a.qscale = (1.0f / sqrtf(float(s.dim))) * kLog2e;
    uintptr_t bits = 0;
    for (const float *y : {x.q, x.k, x.v, x.k_draft, x.v_draft, const_cast<const float *>(x.out)})
        bits |= reinterpret_cast<uintptr_t>(y);
    const bool vec = s.dim % 4 == 0 && (bits & 15u) == 0;
    if (s.dim <= 64) return p.two ? launch<64, 2>(stream, a, vec) : launch<64, 1>(stream, a, vec);
    return p.two ? launch<128, 2>(stream, a, vec) : launch<128, 1>(stream, a, vec);
}

}  // namespace hipk
}  // namespace jade
