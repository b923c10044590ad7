// Paged attention (attention_paged.hip) of many rows on bf16 parts: every FP32 operand is
// held exactly as three bf16 parts and multiplied as six products of parts with FP32 sums
// (split_bf16.hpp), on 32x32x16 MFMAs in the transposed form of attention_flash.hip:
//   S^T[key, row] = sum_d K[key, d] Q[row, d],  O^T[d, row] += sum_key V^T[d, key] P^T[key, row].
// A block has 128 rows (dims to 64) or 256 of a kv head; its waves share tiles of 32 keys,
// whose K and V are split into parts once and staged in LDS, and have 32 rows each. Two
// waves a SIMD, so that one's softmax runs beside the other's MFMAs.
//
// The 16 keys of half a tile lie in one page; each wave stages keys of one half, from a
// descriptor of its own, looked up three tiles ahead. What lies past the last token or in no
// page reads as zeros and is masked. All tiles of all (sequence, kv head, row block)s in a
// row are cut into equal runs, one a block, so that few long sequences fill the chip, too;
// rows come by query, and a block's tiles end where its last query does.
//
// What bounds it: the bf16 matrix cores (66% of the SIMDs' cycles), beside them the softmax
// and the splitting on the VALU, and the clocks that such a load leaves. 512 new tokens over
// 16384 keys, 32 heads (8 of keys) of 128: 657 to 723 us by the card's clocks, 206 to 187
// TFLOP/s; a prompt of 8192 tokens 3099 us (4271 with every row block's tiles counted alike).
// Few rows leave its waves idle: a tile takes one its scores, softmax and outputs one after the
// other, 2.9 us at 128 dims for 48 rows, 3.5 for 128, 5.9 for 256.
//
// V is scaled before it is split and the sums are scaled back, Q is scaled up and K down, so
// every finite V and Q is carried exactly. What the parts do not carry is noticed and done
// again from global memory with FP32 MFMAs, per wave: sums that are not finite (also where a
// later token's value that is not finite met a weight of zero) and queries past 2^64. Sums
// of finite values that FP32 does not hold are taken once more at the end (sum_again).
#include "attention_paged.hpp"
#include "kernels.hpp"
#include "split_bf16.hpp"

namespace jade {
namespace hipk {
namespace {

using namespace paged;
using namespace split;

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kKeys = int(kPagedFlashTile);
// Tiles after which a wave's sums are put aside and begun anew: FP32 sums of 2^22 equal
// weights were off by up to 2.9e-3.
constexpr int kPiece = 128;
// Scaled Q past this takes the FP32 path: then no product of a part of Q with a part of a
// tiny K loses more than an FP32 score's rounding.
constexpr float kMostQ = 0x1p64f * kScaleQ;

__device__ inline float halves_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float halves_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int DP>
struct Shape {
    static constexpr int kWaves = DP <= 64 ? 4 : 8;
    static constexpr int kRows = 32 * kWaves;
    static constexpr int kWide = DP <= 64 ? 64 : 128;            // dims staged (padding reads zero)
    static constexpr int kSteps = DP / 16, kBlocks = DP / 32;    // score steps, output blocks
    static constexpr uint32_t kPartK = kKeys * kWide * 2, kPartV = kWide * kKeys * 2;
    static constexpr uint32_t kTileK = kParts * kPartK, kTileV = kParts * kPartV;
    static constexpr uint32_t kTiles = 2 * (kTileK + kTileV);
    // Q's third part lives in LDS at head dim 128.
    static constexpr bool kQInLds = DP == 128;
    static constexpr uint32_t kLdsBytes = kTiles + (kQInLds ? uint32_t(kWaves) * kSteps * 1024u : 0u);
    static_assert(kLdsBytes <= 160 * 1024, "LDS of a CU");
    static_assert(kKeys * kWide / 8 == 64 * kWaves, "a thread stages eight dims of K");
};

__device__ inline uint32_t dim_now(const PagedArgs &a) {
    uint32_t dim = a.dim;
    asm volatile("" : "+s"(dim));
    return dim;
}

template <int DP>
__global__ __launch_bounds__(64 * Shape<DP>::kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void
attention_paged_flash(PagedArgs a) {
    using S = Shape<DP>;
    constexpr int NW = S::kWaves, KS = S::kSteps, NB = S::kBlocks, WIDE = S::kWide, RB = S::kRows;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, c = lane & 31;
    const uint32_t half = uint32_t(wave) / (NW / 2);  // of a tile's keys, that this wave stages

    // Staging. K: row tid / (WIDE / 8) of a tile, eight dims. V: two dims of four keys.
    const uint32_t row_bytes = a.p_row * 4u;
    const int krow = tid / (WIDE / 8), kq = tid % (WIDE / 8);
    uint32_t koff[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const uint32_t d = 8 * kq + 4 * x;
        koff[x] = d < a.dim ? uint32_t(krow & 15) * row_bytes + d * 4u : kDeadOffset;
    }
    auto swz_k = [](int row) { return WIDE == 128 ? row & 15 : (row >> 1) & 7; };
    const uint32_t kwrite = uint32_t(krow * WIDE * 2 + ((kq ^ swz_k(krow)) << 4));
    // LDS row of V dim 2l + j: the even dims, then the odd ones (so a wave's writes go to
    // adjacent rows and a lane ends up with adjacent dims), dims past DP after them. Chunk
    // 2s + x of a row holds keys 16s + 4x + {0-3, 8-11}: the keys whose weights a lane of half
    // x holds.
    const int vl = WIDE == 128 ? lane : c, vq = WIDE == 128 ? wave : 2 * wave + h;  // dim pair; quad of keys
    const int vs = vq >> 2, vx = vq & 1, vhalf = (vq >> 1) & 1;
    const int vrow = vl < DP / 2 ? vl : DP / 2 + vl;  // dims past DP: rows DP + l - DP / 2 on
    const int vstep = vl < DP / 2 ? DP / 2 : (WIDE - DP) / 2;
    const uint32_t voff = 2 * vl < int(a.dim) ? uint32_t(4 * vx + 8 * vhalf) * row_bytes + uint32_t(8 * vl) : kDeadOffset;
    uint32_t vwrite[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = vrow + j * vstep;
        vwrite[j] = 2 * S::kTileK + uint32_t(row * 64 + (((2 * vs + vx) ^ ((row >> 2) & 3)) << 4) + 8 * vhalf);
    }
    f32x4 kraw[2];
    f32x2 vraw[4];
    auto load_k = [&](__amdgpu_buffer_rsrc_t from, int x) {
        kraw[x] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, int(koff[x]), 0, 0));
    };
    auto load_v = [&](__amdgpu_buffer_rsrc_t from, int e) {
        vraw[e] = __builtin_bit_cast(
            f32x2, __builtin_amdgcn_raw_buffer_load_b64(from, int(voff + uint32_t(e) * row_bytes), 0, 0));
    };
    // Conversion: K pair u, V pair (column j, u), in three pieces.
    uint32_t kparts[kParts][4], vparts[2][kParts][2];
    f32x2 rest;
    auto piece_of = [&](uint32_t &out, int piece, f32x2 x) {
        const f32x2 from = piece == 0 ? x : rest;
        out = pack(from.x, from.y);
        if (piece < 2) rest = rest_of(from, out);
    };
    auto convert_k = [&](int u, int piece) {
        const f32x4 k = kraw[u >> 1];
        piece_of(kparts[piece][u], piece, (u & 1 ? f32x2{k.z, k.w} : f32x2{k.x, k.y}) * kScaleK);
    };
    auto convert_v = [&](int j, int u, int piece) {
        const f32x2 k0 = vraw[2 * u], k1 = vraw[2 * u + 1];
        piece_of(vparts[j][piece][u], piece, (j ? f32x2{k0.y, k1.y} : f32x2{k0.x, k1.x}) * kScaleV);
    };
    auto write_k = [&](int p, uint32_t buf) {
        *reinterpret_cast<u32x4 *>(lds + (kwrite + buf * S::kTileK) + uint32_t(p) * S::kPartK) =
            u32x4{kparts[p][0], kparts[p][1], kparts[p][2], kparts[p][3]};
    };
    auto write_v = [&](int j, int p, uint32_t buf) {
        *reinterpret_cast<u32x2 *>(lds + (vwrite[j] + buf * S::kTileV) + uint32_t(p) * S::kPartV) =
            u32x2{vparts[j][p][0], vparts[j][p][1]};
    };
    // Operand reads.
    uint32_t kread[KS], vread[2];
#pragma unroll
    for (int s = 0; s < KS; ++s) kread[s] = uint32_t(c * WIDE * 2 + (((2 * s + h) ^ swz_k(c)) << 4));
#pragma unroll
    for (int s = 0; s < 2; ++s) vread[s] = 2 * S::kTileK + uint32_t(c * 64 + (((2 * s + h) ^ ((c >> 2) & 3)) << 4));
    bf16x8 kf[2][kParts], q2[2], qp[KS][kParts];
    const uint32_t qplace = S::kTiles + uint32_t(wave * KS * 64 + lane) * 16u;  // third part, kQInLds
    auto read_k = [&](int s, int p, uint32_t buf) {
        kf[s & 1][p] = *reinterpret_cast<const bf16x8 *>(lds + (kread[s] + buf * S::kTileK) + uint32_t(p) * S::kPartK);
    };
    auto read_q = [&](int s) {
        if (S::kQInLds) q2[s & 1] = *reinterpret_cast<const bf16x8 *>(lds + qplace + uint32_t(s) * 1024u);
    };
    auto q_part = [&](int s, int p) { return S::kQInLds && p == 2 ? q2[s & 1] : qp[s][p]; };
    auto publish = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    const Work<kKeys, RB> work(a);
    const uint32_t chunk = (work.total + a.runs - 1) / a.runs;
    const uint32_t run = run_of(blockIdx.x, a.runs);
    uint32_t b, before;
    const uint32_t t_stop = work.start(run + 1, chunk, b, before);
    uint32_t at = work.start(run, chunk, b, before);
    bool odd = false;  // met a sum that is not finite, of weights that are numbers
    while (at < t_stop) {
        const Sequence seq = work.anew(b);
        if (!work.active(seq)) {
            ++b;
            continue;
        }
        const uint32_t all = uniform(work.all_of(seq));
        const Spot spot = work.spot(seq, all, at - before);
        const uint32_t kv = spot.kv, rb = spot.rb, begin = spot.tile, end = min(spot.tiles, begin + (t_stop - at));
        const bool whole = begin == 0 && end == spot.tiles;
        const uint32_t rows = min(uint32_t(RB), seq.count * a.group - rb * RB);
        // Tokens of the block's last query, of this wave's first and last, and of row c's.
        const int old = int(seq.length) - int(seq.count), newest = int(seq.length) - 1;
        const uint32_t r0 = rb * RB + uint32_t(wave) * 32u;
        const int last = min(newest, old + int((rb * RB + RB - 1) / a.group));
        const int low = old + int(r0 / a.group), high = min(newest, old + int((r0 + 31) / a.group));
        const int token = old + int((r0 + uint32_t(c)) / a.group);
        const bool some = uint32_t(wave) * 32u < rows;
        const int t0 = int(begin), t_end = last < 0 ? 0 : int(end);

        // The table's entries for both halves of tile t, -1 past the last; and the keys or
        // values that this wave stages: zeros where they have no page.
        struct Entries {
            float x[2];
        };
        auto entries_of = [&](int t) __attribute__((always_inline)) {
            Args *const now = args_now();
            const float *const table = now->tables + size_t(b) * now->table;
            Entries e;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t n = 2 * uint32_t(t) + s;
                e.x[s] = t < t_end && n * 16 < seq.length ? table[place_of(*now, n).entry] : -1.f;
            }
            return e;
        };
        // Two bits a tile, from this one on: halves without a page. Those past the last token
        // are masked as later than every query.
        uint32_t gaps = 0;
        __amdgpu_buffer_rsrc_t kfrom, vfrom;
        auto take = [&](const Entries &e, int t, int from_now) __attribute__((always_inline)) {
            Args *const now = args_now();
            const uint32_t p0 = uniform(page_of(*now, e.x[0])), p1 = uniform(page_of(*now, e.x[1]));
            gaps |= (uint32_t(p0 == kNoPage) | uint32_t(p1 == kNoPage) << 1) << (2 * from_now);
            const uint32_t n = 2 * uint32_t(t) + half, page = half ? p1 : p0;
            const bool there = page != kNoPage;
            const size_t from = there ? page * now->p_page + kv * now->p_head + size_t(place_of(*now, n).step) * 16 * now->p_row : 0;
            const int bytes = there ? int((min(seq.length - n * 16, 16u) - 1) * now->p_row + now->dim) * 4 : 0;
            kfrom = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(now->k + from), 0, bytes, int(kRawBuffer));
            vfrom = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(now->v + from), 0, bytes, int(kRawBuffer));
        };

        f32x16 acc[NB];
#pragma unroll
        for (int x = 0; x < NB; ++x) acc[x] = f32x16{};
        float row_max = -INFINITY, row_sum = 0.f;  // row_sum: this lane's half of the keys
        float most_q = 0.f;                        // largest |Q| scaled; NaN shows in the sums
        // Row c's place in the block; false past the last.
        struct Row {
            uint32_t mine, query, member;
            bool me;
        };
        auto row_now = [&]() __attribute__((always_inline)) {
            const uint32_t mine = r0 + uint32_t(lane_now() & 31), query = mine / a.group;
            return Row{mine, query, mine - query * a.group, mine - rb * RB < rows};
        };
        const size_t q_base = size_t(b) * a.q_batch + size_t(kv) * a.group * a.q_head;
        // This lane's outputs by four neighbouring dims, first_dim + d and on, each become
        // f(d, x). LDS row r of V is dim 2r (r < DP / 2) or 2 (r - DP / 2) + 1, and
        // a lane holds rows 32x + 8 (v >> 2) + 4h + (v & 3): r, r + 1 and their odd partners are four
        // adjacent dims.
        auto each_four = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll
            for (int y = 0; y < NB * 16; y += 2) {
                const int x = y / 16, v = y % 16, r = 32 * x + 8 * (v >> 2) + (v & 3);
                if (r >= DP / 2) continue;
                const int r2 = r + DP / 2, x2 = r2 / 32, v2 = 4 * (r2 % 32 / 8) + r2 % 4;
                const f32x4 four = f(2 * r, f32x4{acc[x][v], acc[x2][v2], acc[x][v + 1], acc[x2][v2 + 1]});
                acc[x][v] = four.x, acc[x2][v2] = four.y, acc[x][v + 1] = four.z, acc[x2][v2 + 1] = four.w;
            }
        };
        // The sums so far of a long unit, in its slot; `later`: on top of what is there already. Then
        // they begin anew. Or (`back`) what is there on top of the sums.
        auto put_aside = [&](bool later, bool back) __attribute__((always_inline)) {
            const Row row = row_now();
            const uint32_t dim = dim_now(a), first_dim = 8u * uint32_t(lane_now() >> 5);
            Args *const now = args_now();
            const size_t slot = (2 * size_t(run) + (begin == 0)) * RB + (row.mine - rb * RB);
            float2 &kept = reinterpret_cast<float2 *>(now->partial + 2 * size_t(now->runs) * RB * kSlotRow<DP>)[slot];
            const float2 old = row.me && later ? kept : float2{-INFINITY, 0.f};
            const float sum = halves_sum(row_sum), from = row_max == -INFINITY ? 0.f : row_max;
            const float weight = __builtin_amdgcn_exp2f(old.x - from);
            if (row.me) {
                float *const to = now->partial + slot * kSlotRow<DP> + first_dim;
                each_four([&](int d, f32x4 x) __attribute__((always_inline)) {
                    __builtin_amdgcn_sched_barrier(0);  // one at a time: the main loop has no registers to spare
                    if (first_dim + d >= dim) return x;
                    f32x4 &there = *reinterpret_cast<f32x4 *>(to + d);
                    if (later) x += weight * there;
                    if (!back) there = x;
                    return x;
                });
            }
            row_sum = fmaf(weight, old.y, sum);
            if (!back) {
                if (row.me && lane_now() < 32) kept = float2{row_max, row_sum};
                __threadfence_block();  // read by the other half of the wave
                row_sum = 0.f;
#pragma unroll
                for (int x = 0; x < NB; ++x) acc[x] = f32x16{};
            } else if (lane_now() >= 32) {
                row_sum = 0.f;  // halves are added up again
            }
        };
        auto new_piece = [&](int t) __attribute__((always_inline)) {
            if (t != t0 && (t - t0) % kPiece == 0) put_aside(t - t0 != kPiece, false);
        };

        if (t0 < t_end) {
            // Q^T operand: step s holds dims 16s + 8h + e of row c, in log2 units. Rows past the
            // last and dims past dim read zero.
            const Row row = row_now();
            const uint32_t dim = dim_now(a), first_dim = 8u * uint32_t(lane_now() >> 5);
            const uint32_t qoff = uint32_t(row.member * a.q_head + size_t(row.query) * a.q_row) * 4u;
            const uint32_t q_bytes = uint32_t((a.group - 1) * a.q_head + size_t(a.queries - 1) * a.q_row + a.dim) * 4u;
            const __amdgpu_buffer_rsrc_t rq =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(a.q + q_base), 0, int(q_bytes), int(kRawBuffer));
            const Entries e0 = entries_of(t0), e1 = entries_of(t0 + 1);
            Entries ahead = entries_of(t0 + 2);
            f32x4 qraw[KS][2];
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint32_t d = first_dim + 16 * s + 4 * x;
                    const uint32_t from = row.me && d < dim ? qoff + d * 4u : kDeadOffset;
                    qraw[s][x] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rq, int(from), 0, 0));
                }
            take(e0, t0, 0);
#pragma unroll
            for (int x = 0; x < 2; ++x) load_k(kfrom, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) load_v(vfrom, e);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4 p[kParts];
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        f32x2 r = f32x2{qraw[s][x][2 * u], qraw[s][x][2 * u + 1]} * (a.qscale * kScaleQ);
                        most_q = fmaxf(most_q, fmaxf(fabsf(r.x), fabsf(r.y)));
#pragma unroll
                        for (int w = 0; w < kParts; ++w) {
                            const uint32_t k = pack(r.x, r.y);
                            p[w][2 * x + u] = k;
                            r = rest_of(r, k);
                        }
                    }
#pragma unroll
                for (int w = 0; w < kParts; ++w) {
                    if (S::kQInLds && w == 2)
                        *reinterpret_cast<u32x4 *>(lds + qplace + uint32_t(s) * 1024u) = p[w];
                    else
                        qp[s][w] = __builtin_bit_cast(bf16x8, p[w]);
                }
            }
            asm volatile("" : "+v"(most_q));  // taken here, not after the loop from the 8 KS values
            take(e1, t0 + 1, 1);
            __syncthreads();  // the last unit's operands are read
#pragma unroll
            for (int x = 0; x < 12; ++x) convert_k(x / 3, x % 3);
#pragma unroll
            for (int p = 0; p < kParts; ++p) write_k(p, uint32_t(t0) & 1u);
#pragma unroll
            for (int x = 0; x < 2; ++x) load_k(kfrom, x);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int x = 0; x < 6; ++x) convert_v(j, x / 3, x % 3);
#pragma unroll
                for (int p = 0; p < kParts; ++p) write_v(j, p, uint32_t(t0) & 1u);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) load_v(vfrom, e);
            publish();

            auto live = [&](int t) { return some && t * kKeys <= high; };
            f32x16 st;  // scores, then weights
            // A wave's scores, softmax and outputs follow each other, and the other wave's matrix
            // work covers its softmax. K of tile t + 1 is converted beside the scores, V beside the
            // outputs, those of tile t + 2 are loaded; the last tile stages nothing.
            auto tile = [&](int t, auto wc, auto gc) __attribute__((always_inline)) {
                constexpr bool WORK = decltype(wc)::value, STAGE = decltype(gc)::value;
                const uint32_t cur = uint32_t(t) & 1u, other = cur ^ 1u;
                if constexpr (STAGE) {
                    take(ahead, t + 2, 2);
                    ahead = entries_of(t + 3);
                }
                f32x16 sn[2] = {};
                if constexpr (WORK) {
                    read_q(0);
                    read_k(0, 2, cur);
                    read_k(0, 0, cur);
                    read_k(0, 1, cur);
                }
                constexpr int kSlots1 = 6 * KS;
                each<kSlots1>([&](auto nc) __attribute__((always_inline)) {
                    constexpr int n = decltype(nc)::value, s = n / 6, p = n % 6;
                    if constexpr (WORK) {
                        __builtin_amdgcn_sched_barrier(0);
                        sn[s & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s & 1][kPartA[p]], q_part(s, kPartB[p]),
                                                                            sn[s & 1], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                        if constexpr (s + 1 < KS && (p & 1) == 0) read_k(s + 1, p == 0 ? 2 : p == 2 ? 0 : 1, cur);
                        if constexpr (s + 1 < KS && p == 1) read_q(s + 1);
                    }
                    constexpr int lo = kFirstEvent<n, 12, kSlots1>, hi = kFirstEvent<n + 1, 12, kSlots1>;
                    each<STAGE ? hi - lo : 0>([&](auto ec) __attribute__((always_inline)) {
                        constexpr int x = lo + decltype(ec)::value;
                        convert_k(x / 3, x % 3);
                        if constexpr (x % 6 == 5) load_k(kfrom, x / 6);
                        if constexpr (x == 11)
#pragma unroll
                            for (int w = 0; w < kParts; ++w) write_k(w, other);
                    });
                    if constexpr (WORK) __builtin_amdgcn_sched_barrier(0);
                });
                bf16x8 pp[2][kParts];
                bf16x8 va[2][kParts];
                constexpr int kPairs = (NB + 1) / 2;
                auto read_pair = [&](int step, int p) {  // step: (key half, pair of blocks)
                    const int s = step / kPairs, x = 2 * (step % kPairs);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (x + j < NB)
                            va[j][p] = *reinterpret_cast<const bf16x8 *>(lds + (vread[s] + cur * S::kTileV) +
                                                                         uint32_t(x + j) * 2048u + uint32_t(p) * S::kPartV);
                };
                if constexpr (WORK) {
                    read_pair(0, 2);
                    read_pair(0, 0);
                    read_pair(0, 1);
                    st = sn[0] + sn[1];
                    if (t * kKeys + kKeys - 1 > low || gaps & 3) {  // wave-uniform
#pragma unroll
                        for (int v = 0; v < 16; ++v) {
                            const int key = t * kKeys + 8 * (v >> 2) + 4 * h + (v & 3);
                            if (key > token || gaps >> (v >> 3) & 1) st[v] = -INFINITY;
                        }
                    }
                    float top = st[0];
#pragma unroll
                    for (int v = 1; v < 16; ++v) top = fmaxf(top, st[v]);
                    top = halves_max(top);
                    const float next_max = top > row_max + kLazyMax ? top : row_max;
                    const float from = next_max == -INFINITY ? 0.f : next_max;
                    const float old_weight = __builtin_amdgcn_exp2f(row_max - from);
                    float lane_sum = 0.f;
                    uint32_t pw[kParts][8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        st[2 * u] = __builtin_amdgcn_exp2f(st[2 * u] - from);
                        st[2 * u + 1] = __builtin_amdgcn_exp2f(st[2 * u + 1] - from);
                        lane_sum += st[2 * u];
                        lane_sum += st[2 * u + 1];
                        f32x2 r = {st[2 * u], st[2 * u + 1]};
#pragma unroll
                        for (int w = 0; w < kParts; ++w) {
                            pw[w][u] = pack(r.x, r.y);
                            r = rest_of(r, pw[w][u]);
                        }
                    }
                    row_sum = row_sum * old_weight + lane_sum;
                    const bool moved = next_max != row_max;
                    row_max = next_max;
                    if (__any(moved)) {
#pragma unroll
                        for (int x = 0; x < NB; ++x) acc[x] *= old_weight;
                    }
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int p = 0; p < kParts; ++p)
                            pp[s][p] = __builtin_bit_cast(
                                bf16x8, u32x4{pw[p][4 * s], pw[p][4 * s + 1], pw[p][4 * s + 2], pw[p][4 * s + 3]});
                }
                // Outputs by pairs of blocks: 12 MFMAs a pair (six for a lone block).
                constexpr int kSlots2 = 24 * kPairs;
                each<kSlots2>([&](auto nc) __attribute__((always_inline)) {
                    constexpr int n = decltype(nc)::value, step = n / 12, p = n % 12 / 2, j = n & 1;
                    constexpr int s = step / kPairs, x = 2 * (step % kPairs) + j;
                    if constexpr (WORK) {
                        __builtin_amdgcn_sched_barrier(0);
                        if constexpr (x < NB)
                            acc[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[j][kPartA[p]], pp[s][kPartB[p]], acc[x], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                        if constexpr (step + 1 < 2 * kPairs) {
                            if constexpr (p == 0 && j == 1) read_pair(step + 1, 2);
                            if constexpr (p == 3 && j == 1) read_pair(step + 1, 1);
                            if constexpr (p == 5 && j == 1) read_pair(step + 1, 0);
                        }
                    }
                    constexpr int lo = kFirstEvent<n, 12, kSlots2 - 4>, hi = kFirstEvent<n + 1, 12, kSlots2 - 4>;
                    each<STAGE ? hi - lo : 0>([&](auto ec) __attribute__((always_inline)) {
                        constexpr int e = lo + decltype(ec)::value, v = e / 6, u = e / 3 % 2, y = e % 3;
                        convert_v(v, u, y);
                        if constexpr (y == 2) {
                            if constexpr (v == 1) {
                                load_v(vfrom, 2 * u);
                                load_v(vfrom, 2 * u + 1);
                            }
                            if constexpr (u == 1)
#pragma unroll
                                for (int w = 0; w < kParts; ++w) write_v(v, w, other);
                        }
                    });
                    if constexpr (WORK) __builtin_amdgcn_sched_barrier(0);
                });
                if constexpr (STAGE) publish();
                gaps >>= 2;
            };
            for (int t = t0; t < t_end - 1; ++t) {
                new_piece(t);
                if (live(t))
                    tile(t, std::true_type{}, std::true_type{});
                else
                    tile(t, std::false_type{}, std::true_type{});
            }
            if (live(t_end - 1)) tile(t_end - 1, std::true_type{}, std::false_type{});
            if (t_end - 1 - t0 > kPiece) put_aside(true, true);
        }

        // What the parts do not carry: see the file's head.
        float total = row_sum * 0.f;
#pragma unroll
        for (int x = 0; x < NB; ++x)
#pragma unroll
            for (int v = 0; v < 16; ++v) total += acc[x][v] * 0.f;
        float unscale = kUnscaleV;
        if (some && __any(most_q > kMostQ || total != 0.f)) {
            unscale = 1.f;
            row_max = -INFINITY;
            row_sum = 0.f;
#pragma unroll
            for (int x = 0; x < NB; ++x) acc[x] = f32x16{};
            const Row row = row_now();
            const uint32_t dim = dim_now(a);
            const int l = lane_now(), c = l & 31, h = l >> 5;
            const float *const qrow = row.me ? a.q + q_base + row.member * a.q_head + size_t(row.query) * a.q_row : nullptr;
            const int t_last = high < 0 ? -1 : min(t_end - 1, high / kKeys);
            for (int t = t0; t <= t_last; ++t) {
                new_piece(t);
                const Entries e = entries_of(t);
                const uint32_t p0 = uniform(page_of(a, e.x[0])), p1 = uniform(page_of(a, e.x[1]));
                // Key x of the tile: its first dim's place in the pools; 0, which is one, and false
                // where there is none.
                auto row_of = [&](int x, bool &there) {
                    const uint32_t n = 2 * uint32_t(t) + uint32_t(x >> 4), page = x >> 4 ? p1 : p0;
                    there = page != kNoPage && uint32_t(t * kKeys + x) < seq.length;
                    return there ? page * a.p_page + kv * a.p_head + (size_t(place_of(a, n).step) * 16 + (x & 15)) * a.p_row : 0;
                };
                bool key_there;
                const float *const key_row = a.k + row_of(c, key_there);
                f32x16 st = {};
                for (int d0 = 0; d0 < DP; d0 += 8) {
                    const f32x4 k = load_dims<true>(key_there ? key_row : nullptr, d0 + 4 * h, dim);
                    const f32x4 q = load_dims<true>(qrow, d0 + 4 * h, dim) * a.qscale;
#pragma unroll
                    for (int y = 0; y < 4; ++y) st = __builtin_amdgcn_mfma_f32_32x32x2f32(k[y], q[y], st, 0, 0, 0);
                }
                const bool masked = t * kKeys + kKeys - 1 > low;
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int key = t * kKeys + 8 * (v >> 2) + 4 * h + (v & 3);
                    if (key > token || (v >> 3 ? p1 : p0) == kNoPage) st[v] = -INFINITY;
                }
                float top = row_max;
#pragma unroll
                for (int v = 0; v < 16; ++v) top = fmaxf(top, st[v]);
                top = halves_max(top);
                const float from = top == -INFINITY ? 0.f : top;
                const float old_weight = __builtin_amdgcn_exp2f(row_max - from);
                float lane_sum = 0.f;
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    st[v] = __builtin_amdgcn_exp2f(st[v] - from);
                    lane_sum += st[v];
                }
                row_sum = row_sum * old_weight + lane_sum;
                row_max = top;
                // Where not every row sees every key: the finite values, then the weight that each
                // row gives to each special one.
#pragma unroll
                for (int x = 0; x < NB; ++x) {
                    acc[x] *= old_weight;
                    const int r = 32 * x + c;
                    const uint32_t d = r < DP / 2 ? 2 * r : 2 * r - DP + 1;
                    for (int k = -1; k < (masked ? 3 : 0); ++k) {
                        f32x16 sums = {};
#pragma unroll
                        for (int v = 0; v < 16; ++v) {
                            bool there;
                            const float value = a.v[row_of(8 * (v >> 2) + 4 * h + (v & 3), there) + min(d, dim - 1)];
                            const float z = there && d < dim ? value : 0.f;
                            const float y = k >= 0 ? is(k, z) : finite(z) || !masked ? z : 0.f;
                            sums = __builtin_amdgcn_mfma_f32_32x32x2f32(y, st[v], sums, 0, 0, 0);
                        }
#pragma unroll
                        for (int v = 0; v < 16; ++v) acc[x][v] += k < 0 ? sums[v] : sums[v] > 0.f ? special(k) : 0.f;
                    }
                }
            }
            if (t_last - t0 >= kPiece) put_aside(true, true);
            const bool sound = finite(halves_sum(row_sum));
#pragma unroll
            for (int x = 0; x < NB; ++x)
#pragma unroll
                for (int v = 0; v < 16; ++v) odd |= sound && !finite(acc[x][v]);
        }

        row_sum = halves_sum(row_sum);
        const Row row = row_now();
        if (row.me) {
            const uint32_t dim = dim_now(a), first_dim = 8u * uint32_t(lane_now() >> 5);
            const float by = unscale / row_sum;
            const size_t slot = (2 * size_t(run) + (begin == 0)) * RB + (row.mine - rb * RB);
            float *const to = whole ? a.out + row_at(a, b, kv, row.mine) : a.partial + slot * kSlotRow<DP>;
            if (!whole && h == 0)
                reinterpret_cast<float2 *>(a.partial + 2 * size_t(a.runs) * RB * kSlotRow<DP>)[slot] = float2{row_max, row_sum};
            each_four([&](int d, f32x4 x) __attribute__((always_inline)) {
                // A row that sees no key is zeros.
                if (first_dim + d < dim)
                    *reinterpret_cast<f32x4 *>(to + first_dim + d) = row_sum == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : x * by;
                return x;
            });
        }
        at += end - begin;
        if (at >= before + all) {
            before += all;
            ++b;
        }
    }
    if (__builtin_expect(__any(odd), 0)) sum_again<kKeys, RB, kSlotRow<DP>, 32, true>();
}

template <int DP>
void launch(hipStream_t stream, const PagedArgs &a) {
    hipLaunchKernelGGL((attention_paged_flash<DP>), dim3(a.runs), dim3(64 * Shape<DP>::kWaves), 0, stream, a);
}

}  // namespace

uint32_t paged_flash_lds_bytes(uint32_t dim) {
    return dim <= 32 ? Shape<32>::kLdsBytes : dim <= 64 ? Shape<64>::kLdsBytes : dim <= 96 ? Shape<96>::kLdsBytes : Shape<128>::kLdsBytes;
}

void launch_paged_flash(hipStream_t stream, const PagedArgs &a) {
    if (a.dim <= 32)
        launch<32>(stream, a);
    else if (a.dim <= 64)
        launch<64>(stream, a);
    else if (a.dim <= 96)
        launch<96>(stream, a);
    else
        launch<128>(stream, a);
}

}  // namespace hipk
}  // namespace jade
