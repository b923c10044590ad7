// Ragged attention (attention_ragged.hip) of more than 16 rows on bf16 parts: every FP32
// operand is held exactly as three bf16 parts and multiplied as six products of parts with
// FP32 sums (split_bf16.hpp), on 32x32x16 MFMAs in the transposed form of
// attention_flash.hip. Head dims are padded to 64, 96 or 128. A wave has all 32 or 64 rows of its block and
// 32 of a tile's 128 keys. Both products take their dims and keys in the order in which
// a lane's 16-byte loads of K and V leave them, so K and V go from memory to registers
// and are split there, by the one wave that multiplies them; LDS has only the parts of
// Q, which the four waves share. A last chunk that is not whole reads into the next row (or
// nothing past the tile): Q's parts are zeros there, and V's dims past the last are dropped.
//
// One wave a SIMD (but for 32 rows of few dims), so it overlaps its own work: an MFMA every 32 cycles, and between
// two of them two of the twelve pieces in which the next eight values of K or V are
// split; a chunk is loaded again, for the next tile, as soon as it is split. For 64
// rows and 32 keys of 128 dims that is 192 MFMAs (6144 cycles of a SIMD; FP32 MFMAs
// take 16384) and 1300 other vector instructions, most of them beside the MFMAs; masks,
// maxima and the first weights are between the two products and beside none. 64 nodes x 32
// heads (8 of keys) over 4 sequences of at most 4096 keys of 128: 115 to 125 us by card, 109
// to 118 TFLOP/s; 13 nodes over 8 sequences: 67 to 74 us, 3.0 to 3.2 TB/s of K and V. No unit
// bounds them: of a wave's time MFMAs take 47 and 38%, vector instructions, most of them
// beside MFMAs, 56 and 49%, waits for memory 16 and 20%, waits to issue 20 and 22%; 23 and
// 30% of the SIMDs' cycles have no wave (unequal runs, the launch's ends). A run's unit costs
// 8 to 11 us besides its tiles: Q's loads and parts, the first tile's loads, the waves' sums
// joined.
//
// Q and V are scaled up and K down before they are split. So every finite Q and V is
// carried exactly (V as it is left nothing of values below 2^-134), and scores are in FP32's
// own range (with K as it is they passed it from 2^104 on, and a score of -inf weighs
// nothing without a trace in the sums). A K below 2^-86 loses less than 2^-110, which moves
// no score by more than 2^-46 a dim: a query is at most 2^64. The scaling is beside the
// MFMAs: in one run 13 nodes as above took 67.3 us without it and with it, 64 nodes 119.1
// and 115.4 (a look at the scores of each tile instead cost 1-2%). What the parts do not
// carry (sums that are not finite, queries past 2^64) the block notices when it joins its
// sums, and does them again with FP32 MFMAs.
#include "kernels.hpp"
#include "ragged_device.hpp"
#include "split_bf16.hpp"

namespace jade {
namespace hipk {
namespace {

using namespace ragged;
using namespace split;

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTile = 128;  // keys per tile, 32 for each wave by keys
constexpr float kMostQ = 0x1p64f * kScaleQ;

__device__ inline float halves_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float halves_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Piece n < 12 of splitting eight values: pairs 0 and 1 in turn, a part at a time, then
// pairs 2 and 3 (a pair's next part waits for its rest, so two pairs take turns);
// pair_of(n) says whose. `rest` holds what is left of the two pairs, at first the pairs
// themselves. Rests by a shift or a mask and a subtraction: v_dot2_f32_bf16, which does
// it in one instruction, waits for the matrix cores (four of them after a 32-cycle MFMA:
// 62 cycles; eight VALU instructions: 42).
constexpr int pair_of(int n) { return n / 6 * 2 + n % 2; }
__device__ inline void split_piece(int n, f32x2 (&rest)[2], uint32_t (&out)[kParts][4]) {
    const int w = n % 6 / 2;
    f32x2 &x = rest[n % 2];
    const uint32_t p = pack(x.x, x.y);
    out[w][pair_of(n)] = p;
    if (w < 2) x = f32x2{x.x - low_part(p), x.y - high_part(p)};
}
__device__ inline bf16x8 part_of(const uint32_t (&p)[kParts][4], int w) {
    return __builtin_bit_cast(bf16x8, u32x4{p[w][0], p[w][1], p[w][2], p[w][3]});
}

// The lane's number, made anew: what is computed from it is not kept in registers from
// outside the main loop.
__device__ inline int lane_now() {
    int l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(l));
    return l;
}

template <int DP, int QG>
struct Shape {
    static constexpr int kRows = 32 * QG, kPitch = DP + 4;
    static constexpr int kSteps = DP / 16;  // score steps
    static constexpr int kOut = DP / 32;    // output blocks of 32 dims: dims kOut * r + e
    // Where K and V of a tile are loaded: each chunk as soon as the last tile's is split,
    // or, where two row groups leave no registers for all of both, V before the scores
    // and K before and amid the outputs.
    static constexpr int kWavesASimd = QG == 1 && DP <= 64 ? 2 : 1;  // what the registers hold
    static constexpr bool kEarly = QG == 1 || DP <= 96;
    static constexpr int kEarlyK = kEarly ? kSteps : 0;
    static_assert(QG * kSteps * kParts * 1024 <= kWaves * kRows * kPitch * 4, "Q's parts fit the sums' space");
};

// QG: groups of 32 rows, all of them every wave's.
template <int DP, int QG, bool VEC>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(Shape<DP, QG>::kWavesASimd, Shape<DP, QG>::kWavesASimd))) void
attention_ragged_parts(RaggedArgs a) {
    using S = Shape<DP, QG>;
    constexpr int KS = S::kSteps, NB = S::kOut, RB = S::kRows;
    typedef float vec __attribute__((ext_vector_type(NB)));
    __shared__ __attribute__((aligned(16))) float part[kWaves][RB][S::kPitch];
    __shared__ float2 ml[kWaves][RB];
    __shared__ RowPlan plans[RB];
    __shared__ uint64_t sees[kMaxTreeNodes][kWords];
    __shared__ int above[kMaxTreeNodes];
    __shared__ float2 seen_so_far[kWaves][QG][64];  // running maximum and sum of a lane's rows
    __shared__ int far;  // a query that the parts do not carry
    char *const qs = reinterpret_cast<char *>(&part[0][0][0]);  // Q's parts until the sums are joined
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t units = a.kv_heads * a.row_blocks;
    const Spread<kTile> spread(a);
    const uint32_t total = spread.total * units, chunk = (total + a.runs - 1) / a.runs;
    const uint32_t run = run_of(blockIdx.x, a.runs);
    uint32_t b, before;
    const uint32_t t_stop = spread.start(run + 1, chunk, units, b, before);
    uint32_t t = spread.start(run, chunk, units, b, before);

    const uint32_t row_bytes = a.k_row * 4u;
    uint32_t tree = ~0u;  // the sequence whose tree is in LDS
    while (t < t_stop) {
        const uint32_t len = spread.length(b);
        const uint32_t cached = (len + kTile - 1) / kTile, tiles = cached + spread.draft_tiles;
        if (!tiles) {
            ++b;
            continue;
        }
        const uint32_t in = t - before * units, unit = in / tiles, begin = in - unit * tiles;
        const uint32_t kv = unit / a.row_blocks, rb = unit - kv * a.row_blocks;
        const uint32_t end = min(tiles, begin + (t_stop - t));
        const bool whole = begin == 0 && end == tiles;
        float above_me = 0.f;
        if (end > cached && tree != b && tid < int(a.nodes)) above_me = a.parents[size_t(b) * a.nodes + tid];

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
        f32x4 kf[KS][2];
        vec vf[2][8];
        struct Offsets {
            uint32_t k, v;
            int last;  // K's chunks of eight dims that have this lane's four of them
        };
        auto offsets = [&]() __attribute__((always_inline)) {
            const uint32_t l = lane_now();
            const uint32_t half = l >> 5, row = l & 31;
            return Offsets{(32 * wave + row) * row_bytes + 16 * half,
                           NB * row < a.dim ? (32 * wave + 4 * half) * row_bytes + 4 * NB * row : kDeadOffset,
                           int((a.dim + 3) / 4 + 1 - half) / 2};
        };
        // Dims of score step s, load x: 8 y + 4 h + 0 .. 3, y = 2 s + x.
        auto load_k = [&](__amdgpu_buffer_rsrc_t from, const Offsets &o, int s) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int y = 2 * s + x;
                const uint32_t at = y < o.last ? o.k + 32u * y : kDeadOffset;
                kf[s][x] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, int(at), 0, 0));
            }
        };
        // Dims NB c .. + NB - 1 of keys 16 s + 4 h + (u & 3) + 8 (u >> 2).
        auto load_v = [&](__amdgpu_buffer_rsrc_t from, uint32_t voff, int s, int u) __attribute__((always_inline)) {
            const uint32_t at = voff + uint32_t(16 * s + (u & 3) + 8 * (u >> 2)) * row_bytes;
            if constexpr (NB == 4)
                vf[s][u] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b128(from, int(at), 0, 0));
            else if constexpr (NB == 3)
                vf[s][u] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b96(from, int(at), 0, 0));
            else
                vf[s][u] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b64(from, int(at), 0, 0));
        };
        // Row r of the block, from its first dim; null past the last row.
        auto q_row = [&](int r) -> const float * {
            const uint32_t at = rb * RB + r, head = at / a.queries, query = at - head * a.queries;
            if (head >= a.group) return nullptr;
            return a.q + size_t(b) * a.q_batch + (size_t(kv) * a.group + head) * a.q_head + size_t(query) * a.q_row;
        };
        // Q first, then the first tile; from there on a chunk is loaded again once it is
        // split. A wave stages every fourth of the QG * KS (row group, step)s.
        constexpr int kItems = (QG * KS + kWaves - 1) / kWaves;
        f32x4 qraw[kItems][2];
        {
            const int l = lane_now();
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                const int n = kWaves * i + wave, r = n / KS, s = n % KS;
                const float *row = r < QG ? q_row(32 * r + (l & 31)) : nullptr;
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    qraw[i][y] = load_dims<VEC>(row, 16 * s + 8 * y + 4 * (l >> 5), a.dim);
            }
            const auto kfrom = tile_of(kb, kd, begin), vfrom = tile_of(vb, vd, begin);
            const Offsets at = offsets();
#pragma unroll
            for (int s = 0; s < KS; ++s) load_k(kfrom, at, s);
            if (S::kEarly)
#pragma unroll
                for (int u = 0; u < 16; ++u) load_v(vfrom, at.v, u >> 3, u & 7);
        }
        // Q's parts: for group r, step s, part w and lane, 16 bytes at ((r KS + s) kParts + w) 64 + lane.
        __syncthreads();  // the last unit's sums are read
        if (tid == 0) far = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int n = kWaves * i + wave, r = n / KS, s = n % KS;
            if (r >= QG) break;
            uint32_t p[kParts][4];
            bool past = false;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const f32x4 q = qraw[i][y] * (a.qscale * kScaleQ);
#pragma unroll
                for (int e = 0; e < 4; ++e) past |= fabsf(q[e]) > kMostQ;
                f32x2 rest[2] = {{q.x, q.y}, {q.z, q.w}};
#pragma unroll
                for (int n = 0; n < 6; ++n) split_piece(6 * y + n, rest, p);
            }
            if (past) far = 1;
#pragma unroll
            for (int w = 0; w < kParts; ++w)
                *reinterpret_cast<bf16x8 *>(qs + (((r * KS + s) * kParts + w) * 64 + lane) * 16) = part_of(p, w);
        }
        if (end > cached && tree != b) {
            see_ancestors(a.nodes, above_me, sees, above);
            tree = b;
        } else {
            __syncthreads();
        }

        f32x16 acc[QG][NB], st[QG];
        float top[QG], sum[QG];  // of the tile at hand; between tiles in LDS, where nothing spills them
        float2 (&state)[QG][64] = seen_so_far[wave];
        auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < QG; ++r) {
                state[r][lane] = float2{-INFINITY, 0.f};
#pragma unroll
                for (int e = 0; e < NB; ++e) acc[r][e] = f32x16{};
            }
        };
        clear();
        // Keys that this wave's rows do not see, of its 32 in tile x.
        auto mask = [&](uint32_t x) __attribute__((always_inline)) {
            if (x < cached && (x + 1) * kTile <= len) return;
            const int l = lane_now(), c = l & 31, h = l >> 5;
            if (x >= cached) {
                const uint32_t key = (x - cached) * kTile + 32 * wave;
#pragma unroll
                for (int r = 0; r < QG; ++r) {
                    const uint32_t node = (rb * RB + 32 * r + c) % a.queries;  // queries == nodes
                    const uint32_t seen = uint32_t(sees[node][key / 64] >> (key & 63)) >> (4 * h);
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (!(seen >> (8 * (v >> 2) + (v & 3)) & 1)) st[r][v] = -INFINITY;
                }
            } else {
                const int first = int(x) * kTile + 32 * wave + 4 * h;
#pragma unroll
                for (int r = 0; r < QG; ++r)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (first + 8 * (v >> 2) + (v & 3) >= int(len)) st[r][v] = -INFINITY;
            }
        };
        // The running maximum of the rows past this tile's scores; what was summed so far
        // is scaled to it.
        auto raise = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < QG; ++r) {
                top[r] = state[r][lane].x;
                sum[r] = state[r][lane].y;
                float most = st[r][0];
#pragma unroll
                for (int v = 1; v < 16; ++v) most = fmaxf(most, st[r][v]);
                if (__any(most > top[r] + kLazyMax)) {
                    const float reached = fmaxf(top[r], halves_max(most));
                    const float keep = reached == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top[r] - reached);
                    top[r] = reached;
                    sum[r] *= keep;
#pragma unroll
                    for (int e = 0; e < NB; ++e) acc[r][e] *= keep;
                }
            }
        };
        auto keep_state = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < QG; ++r) state[r][lane] = float2{top[r], sum[r]};
        };
        // Score v of row group r to its weight.
        auto weigh = [&](int r, int v) __attribute__((always_inline)) {
            const float weight = __builtin_amdgcn_exp2f(st[r][v] - (top[r] == -INFINITY ? 0.f : top[r]));
            sum[r] += weight;
            return weight;
        };

        // Two buffers of parts each for K steps, Q steps and V octets (s, e): one is
        // multiplied while the next is made.
        uint32_t kp[2][kParts][4], vp[2][kParts][4];
        bf16x8 q0[2][QG], q12[QG][2];  // a step's last product takes Q's part 0, so that one twice
        f32x2 rest[2];
        auto read_q = [&](int s, int w) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < QG; ++r)
                (w ? q12[r][w - 1] : q0[s & 1][r]) =
                    *reinterpret_cast<const bf16x8 *>(qs + (((r * KS + s) * kParts + w) * 64 + lane) * 16);
        };
        // What is split beside the products of a tile, in order: K's steps 1 .. KS - 1, V's
        // octets (o: keys 16 (o / NB) .. + 15 of the lane's half, dim o % NB) and the next
        // tile's K step 0.
        auto values = [&](int q, int pair) __attribute__((always_inline)) {
            const int s = (q + 1) % (KS + 2 * NB), o = s - KS;
            if (s < KS) {
                const f32x4 k = kf[s][pair / 2] * kScaleK;
                return pair % 2 ? f32x2{k.z, k.w} : f32x2{k.x, k.y};
            }
            return f32x2{vf[o / NB][2 * pair][o % NB], vf[o / NB][2 * pair + 1][o % NB]} * kScaleV;
        };
        auto split = [&](int q, int n) __attribute__((always_inline)) {
            const int s = (q + 1) % (KS + 2 * NB), o = s - KS;
            split_piece(n, rest, s < KS ? kp[s & 1] : vp[o & 1]);
            if (n % 6 >= 4) rest[n % 2] = n < 6 ? values(q, pair_of(n + 2)) : values((q + 1) % (KS + 2 * NB), pair_of(n - 10));
        };
#pragma unroll
        for (int n = 0; n < 2; ++n) rest[n] = values(KS + 2 * NB - 1, n);
#pragma unroll
        for (int n = 0; n < 12; ++n) split(KS + 2 * NB - 1, n);
#pragma unroll
        for (int w = 0; w < kParts; ++w) read_q(0, w);
        auto kfrom = tile_of(kb, kd, begin + 1), vfrom = tile_of(vb, vd, S::kEarly ? begin + 1 : begin);
        Offsets at = offsets();

        for (uint32_t x = begin; x < end; ++x) {
#pragma unroll
            for (int r = 0; r < QG; ++r) st[r] = f32x16{};
            each<6 * KS * QG>([&](auto nc) __attribute__((always_inline)) {
                constexpr int i = decltype(nc)::value % (6 * QG), s = decltype(nc)::value / (6 * QG), p = i / QG, r = i % QG;
                __builtin_amdgcn_sched_barrier(0);
                st[r] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    part_of(kp[s & 1], kPartA[p]), kPartB[p] ? q12[r][kPartB[p] - 1] : q0[s & 1][r], st[r], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                each<2 / QG>([&](auto ec) __attribute__((always_inline)) { split(s, 2 * i / QG + decltype(ec)::value); });
                if constexpr (s + 1 < KS && r == QG - 1) {
                    // Each part once its last product is issued (B's parts go 0 2 1 0 1 0).
                    if constexpr (p == 0) read_q(s + 1, 0);
                    if constexpr (p == 1) read_q(s + 1, 2);
                    if constexpr (p == 4) read_q(s + 1, 1);
                }
                // Step s's values are split: K's next tile there.
                if constexpr (p == 0 && r == QG - 1 && s < S::kEarlyK) load_k(kfrom, at, s);
                // V's rows where they are not loaded yet: the first eight early.
                if constexpr (!S::kEarly && r == QG - 1) {
                    constexpr int n = 6 * s + p, last = 6 * KS - 6;
                    if constexpr (n % 2 == 1 && n < 16) load_v(vfrom, at.v, 0, n / 2);
                    if constexpr (n >= 16 && (n - 16) % ((last - 16) / 8) == 0 && (n - 16) / ((last - 16) / 8) < 8)
                        load_v(vfrom, at.v, 1, (n - 16) / ((last - 16) / 8));
                }
            });
            __builtin_amdgcn_sched_barrier(0);
            mask(x);
            raise();
            // Weights and their parts, of keys 0 .. 15 here, of 16 .. 31 beside the first outputs.
            uint32_t pp[QG][2][kParts][4];
            f32x2 prest[2];
            auto split_p = [&](int r, int s, int n) __attribute__((always_inline)) {
                const int v = 8 * s + 2 * pair_of(n);
                if (n % 6 < 2) prest[n % 2] = f32x2{weigh(r, v), weigh(r, v + 1)};
                split_piece(n, prest, pp[r][s]);
            };
#pragma unroll
            for (int r = 0; r < QG; ++r)
#pragma unroll
                for (int n = 0; n < 12; ++n) split_p(r, 0, n);
            each<12 * NB * QG>([&](auto nc) __attribute__((always_inline)) {
                constexpr int n = decltype(nc)::value, i = n % (6 * QG), o = n / (6 * QG), p = i / QG, r = i % QG;
                constexpr int s = o / NB, e = o % NB;
                __builtin_amdgcn_sched_barrier(0);
                acc[r][e] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(part_of(vp[o & 1], kPartA[p]),
                                                                    part_of(pp[r][s], kPartB[p]), acc[r][e], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                constexpr int lo = kFirstEvent<n, 12 * QG, 6 * NB * QG>, hi = kFirstEvent<n + 1, 12 * QG, 6 * NB * QG>;
                if constexpr (o < NB)
                    each<hi - lo>([&](auto ec) __attribute__((always_inline)) {
                        constexpr int j = lo + decltype(ec)::value;
                        split_p(j / 12, 1, j % 12);
                    });
                if constexpr (n == 6 * NB * QG) keep_state();
                each<2 / QG>([&](auto ec) __attribute__((always_inline)) { split(KS + o, 2 * i / QG + decltype(ec)::value); });
                if constexpr (r == QG - 1) {
                    // The last octet of 16 keys is split from octet NB - 2's products on: V's
                    // next tile there, or K's remaining steps.
                    constexpr int u = 6 * (o % NB - (NB - 1)) + p;  // slots since
                    if constexpr (S::kEarly && (u == 0 || u == 1 || u == 2 || u == 3))
#pragma unroll
                        for (int j = 2 * u; j < 2 * u + 2; ++j) load_v(vfrom, at.v, s, j);
                    constexpr int at0 = 6 * o + p;
                    if constexpr (!S::kEarly && at0 % 2 == 1 && at0 < KS) load_k(kfrom, at, at0 / 2);
                    if constexpr (!S::kEarly && s == 0 && u >= 0 && u < KS / 2) load_k(kfrom, at, KS / 2 + u);
                    if constexpr (o + 1 == 2 * NB && p < kParts) read_q(0, p);
                    // The tile after the next.
                    if constexpr (n / QG == 12 * NB - 1) {
                        kfrom = tile_of(kb, kd, x + 2);
                        vfrom = tile_of(vb, vd, S::kEarly ? x + 2 : x + 1);
                        at = offsets();
                    }
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        }

        // The sums of a wave to LDS: dim NB i + e of row c for i = 8 (v >> 2) + 4 h + (v & 3).
        auto hand_over = [&]() __attribute__((always_inline)) {
            const int l = lane_now(), c = l & 31, h = l >> 5;
            __syncthreads();
#pragma unroll
            for (int r = 0; r < QG; ++r) {
                const float2 mine = state[r][lane];
                const float all = halves_sum(mine.y);
                if (h == 0) ml[wave][32 * r + c] = float2{mine.x, all};
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    vec o;
#pragma unroll
                    for (int e = 0; e < NB; ++e) o[e] = acc[r][e][v];
                    float *const to = &part[wave][32 * r + c][NB * (8 * (v >> 2) + 4 * h + (v & 3))];
                    if constexpr (NB == 3)  // twelve bytes
#pragma unroll
                        for (int e = 0; e < NB; ++e) to[e] = o[e];
                    else
                        *reinterpret_cast<vec *>(to) = o;
                }
            }
            __syncthreads();
        };
        hand_over();
        if (finish<DP, RB, VEC>(a, run, b, kv, rb, whole, begin == 0, part, ml, plans, sees, kUnscaleV)) far = 1;
        __syncthreads();
        if (far) {  // what the parts do not carry: see the file's head
            clear();
            const int l = lane_now(), c = l & 31, h = l >> 5;
            for (uint32_t x = begin; x < end; ++x) {
                const bool drafted = x >= cached;
                const uint32_t tile = drafted ? x - cached : x, keys = drafted ? a.nodes : len;
                const uint32_t key0 = tile * kTile + 32 * wave;
                const float *krow = (drafted ? kd : kb) + size_t(key0 + c) * a.k_row;
                const float *vrow = (drafted ? vd : vb) + size_t(key0) * a.k_row;
#pragma unroll
                for (int r = 0; r < QG; ++r) {
                    st[r] = f32x16{};
                    const float *qrow = q_row(32 * r + c);
                    for (int d0 = 0; d0 < DP; d0 += 8) {
                        const int d = d0 + 4 * h;
                        const f32x4 q = load_dims<VEC>(qrow, d, a.dim) * a.qscale;
                        const f32x4 k = load_dims<VEC>(key0 + c < keys ? krow : nullptr, d, a.dim);
#pragma unroll
                        for (int e = 0; e < 4; ++e) st[r] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[e], st[r], 0, 0, 0);
                    }
                }
                mask(x);
                raise();
#pragma unroll
                for (int r = 0; r < QG; ++r)
#pragma unroll
                    for (int v = 0; v < 16; ++v) st[r][v] = weigh(r, v);
                keep_state();
                // Drafted values that are not finite, which not every row may see: the finite
                // ones, then the weight that each row gives to each special one.
                for (int e = 0; e < NB; ++e)
                    for (int k = -1; k < (drafted ? 3 : 0); ++k)
#pragma unroll
                        for (int r = 0; r < QG; ++r) {
                            f32x16 sums = {};
#pragma unroll
                            for (int v = 0; v < 16; ++v) {
                                const uint32_t key = 8 * (v >> 2) + 4 * h + (v & 3);
                                const int d = NB * c + e;
                                const float z = d < a.dim && key0 + key < keys ? vrow[size_t(key) * a.k_row + d] : 0.f;
                                const float y = k >= 0 ? is(k, z) : finite(z) || !drafted ? z : 0.f;
                                sums = __builtin_amdgcn_mfma_f32_32x32x2f32(y, st[r][v], sums, 0, 0, 0);
                            }
#pragma unroll
                            for (int v = 0; v < 16; ++v) {
                                const float more = k < 0 ? sums[v] : sums[v] > 0.f ? special(k) : 0.f;
#pragma unroll
                                for (int f = 0; f < NB; ++f)
                                    if (f == e) acc[r][f][v] += more;
                            }
                        }
            }
            hand_over();
            finish<DP, RB, VEC>(a, run, b, kv, rb, whole, begin == 0, part, ml, plans, sees, 1.f);
        }
        t += end - begin;
        if (t >= (before + tiles) * units) {
            before += tiles;
            ++b;
        }
    }
}

template <int DP, int QG, bool VEC>
void launch(hipStream_t stream, const RaggedArgs &a) {
    hipLaunchKernelGGL((attention_ragged_parts<DP, QG, VEC>), dim3(a.runs), dim3(kThreads), 0, stream, a);
}

template <int DP, int QG>
void launch_rows(hipStream_t stream, const RaggedArgs &a) {
    a.dim % 4 ? launch<DP, QG, false>(stream, a) : launch<DP, QG, true>(stream, a);
}

}  // namespace

uint32_t ragged_parts_lds_bytes(uint32_t dim, uint32_t block_rows) {
    const uint32_t pitch = (dim <= 64 ? 64 : dim <= 96 ? 96 : 128) + 4;
    return uint32_t(kWaves * block_rows * (pitch * sizeof(float) + sizeof(float2)) + block_rows * sizeof(RowPlan) +
                    kMaxTreeNodes * (kWords * sizeof(uint64_t) + sizeof(int)) +
                    kWaves * block_rows / 32 * 64 * sizeof(float2) + sizeof(int));
}

void launch_ragged_parts(hipStream_t stream, const RaggedArgs &a, uint32_t block_rows) {
    if (a.dim <= 64)
        block_rows == 32 ? launch_rows<64, 1>(stream, a) : launch_rows<64, 2>(stream, a);
    else if (a.dim <= 96)
        block_rows == 32 ? launch_rows<96, 1>(stream, a) : launch_rows<96, 2>(stream, a);
    else
        block_rows == 32 ? launch_rows<128, 1>(stream, a) : launch_rows<128, 2>(stream, a);
}

}  // namespace hipk
}  // namespace jade
