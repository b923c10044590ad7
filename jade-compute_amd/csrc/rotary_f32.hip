// Rotary positions, alone or after an RMS norm of every head, over tensors of
// heads laid out [batch, seq, heads, dim] or [batch, heads, seq, dim], from
// either layout into either:
//   y = x                                   (rotary)
//   y = x * rsqrt(mean(x^2) + eps) * weight (qk_norm_rotary, over a head)
//   out_a = m (y_a cos t - y_b sin t), out_b = m (y_b cos t + y_a sin t)
// for the pairs (a, b) = (i, i + R/2) or (2i, 2i + 1), i < R/2, of the first R
// dims, t = 2 pi * position * rate_i; the dims from R on are copied. The
// inverse negates the sine: the transposed map, so the gradient too.
//
// The angle: position * rate in 64 bits, in turns, reduced there to within an
// eighth of a turn of a multiple of a quarter; only that remainder goes to FP32
// (off by at most 2^-25 of itself), into Taylor series (FP32 angles are off by
// 2^-24 of the whole angle: 0.06 at position 10^6).
#include "kernels.hpp"

namespace jade {
namespace hipk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr uint32_t kMaxBlocks = 1u << 20;

// cos and sin of `turns` full turns. On |x| <= pi/4 the first terms left out
// are x^11/11! < 1.8e-9 of sin x and x^12/12! < 1.2e-10.
__device__ inline void turn(double turns, float &cosine, float &sine) {
    const double part = turns - floor(turns), quarter = rint(part * 4.0);
    const float x = float((part - quarter * 0.25) * 6.283185307179586476925286766559);
    const int which = int(quarter);
    const float z = x * x;
    const float s = x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), 1.f);
    const float c =
        fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
    const float a = which & 1 ? s : c, b = which & 1 ? c : s;
    cosine = (which + 1) & 2 ? -a : a;
    sine = which & 2 ? -b : b;
}

// Offset of (batch b, token s, head h) in a tensor of `heads` heads.
__device__ inline size_t head_at(const RotaryArgs &a, bool token_major, uint32_t heads, uint32_t b, uint32_t s,
                                 uint32_t h) {
    return (token_major ? (size_t(b) * a.seq + s) * heads + h : (size_t(b) * heads + h) * a.seq + s) * a.dim;
}

struct Head {
    const float *x, *weight;
    float *out;
};
// Head h of the first tensor, or of the second from a.heads on.
__device__ inline Head head_of(const RotaryArgs &a, uint32_t b, uint32_t s, uint32_t h) {
    const bool second = h >= a.heads;
    const uint32_t heads = second ? a.heads2 : a.heads, at = second ? h - a.heads : h;
    return {(second ? a.x2 : a.x) + head_at(a, a.token_major, heads, b, s, at), second ? a.weight2 : a.weight,
            (second ? a.out2 : a.out) + head_at(a, a.out_token_major, heads, b, s, at)};
}

// Heads whose rows take whole float4s: LANES lanes (a power of two) share a head,
// a lane with eight of its dims: four pairs, or eight dims that are not turned.
// A wave keeps one token's angles and goes over `per_wave` groups of 64 / LANES
// heads.
template <int LANES, bool NORM>
__global__ __launch_bounds__(kThreads) void rotary_lanes(RotaryArgs a, uint32_t per_wave, uint32_t spans,
                                                         uint32_t items) {
    const int lane = threadIdx.x & 63, unit = lane % LANES;
    const uint32_t all = a.heads + a.heads2, turned = a.rotary_dim / 8;
    const bool mine = uint32_t(unit) < a.dim / 8, turns = uint32_t(unit) < turned;
    const uint32_t d0 = a.interleaved || !turns ? 8 * unit : 4 * unit;
    const uint32_t d1 = a.interleaved || !turns ? d0 + 4 : d0 + a.rotary_dim / 2;
    for (uint32_t item = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); item < items;
         item += gridDim.x * (kThreads / 64)) {
        const uint32_t token = item / spans, h0 = item % spans * per_wave * (64 / LANES);
        const uint32_t b = token / a.seq, s = token % a.seq;
        f32x4 c = {1.f, 1.f, 1.f, 1.f}, sn = {0.f, 0.f, 0.f, 0.f};
        if (turns) {
            const double position = a.positions[token];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float cosine, sine;
                turn(position * a.rates[4 * unit + e], cosine, sine);
                c[e] = cosine * a.magnitude;
                sn[e] = a.inverse ? -sine * a.magnitude : sine * a.magnitude;
            }
        }
        for (uint32_t i = 0; i < per_wave; ++i) {
            const uint32_t h = h0 + i * (64 / LANES) + lane / LANES;
            const bool live = h < all && mine;
            if (!NORM && !live) continue;
            const Head head = head_of(a, b, s, h < all ? h : 0);
            f32x4 x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0;
            if (live) {
                x0 = *reinterpret_cast<const f32x4 *>(head.x + d0);
                x1 = *reinterpret_cast<const f32x4 *>(head.x + d1);
            }
            if constexpr (NORM) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) sum = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], sum));
#pragma unroll
                for (int offset = LANES / 2; offset > 0; offset >>= 1) sum += __shfl_xor(sum, offset);
                if (!live) continue;
                const float inv = rsqrtf(sum / float(a.dim) + a.epsilon);
                x0 = x0 * inv * *reinterpret_cast<const f32x4 *>(head.weight + d0);
                x1 = x1 * inv * *reinterpret_cast<const f32x4 *>(head.weight + d1);
            }
            f32x4 y0 = x0, y1 = x1;
            if (turns) {
                if (a.interleaved) {
                    y0 = {x0.x * c.x - x0.y * sn.x, x0.y * c.x + x0.x * sn.x, x0.z * c.y - x0.w * sn.y,
                          x0.w * c.y + x0.z * sn.y};
                    y1 = {x1.x * c.z - x1.y * sn.z, x1.y * c.z + x1.x * sn.z, x1.z * c.w - x1.w * sn.w,
                          x1.w * c.w + x1.z * sn.w};
                } else {
                    y0 = x0 * c - x1 * sn;
                    y1 = x1 * c + x0 * sn;
                }
            }
            *reinterpret_cast<f32x4 *>(head.out + d0) = y0;
            *reinterpret_cast<f32x4 *>(head.out + d1) = y1;
        }
    }
}

// Any other head: one wave a head, pairs and single dims in turn.
template <bool NORM>
__global__ __launch_bounds__(kThreads) void rotary_any(RotaryArgs a, uint32_t per_wave, uint32_t spans,
                                                       uint32_t items) {
    constexpr int kPairs = int(kMaxRotaryDim) / 2 / 64;
    const int lane = threadIdx.x & 63;
    const uint32_t all = a.heads + a.heads2, pairs = a.rotary_dim / 2;
    for (uint32_t item = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); item < items;
         item += gridDim.x * (kThreads / 64)) {
        const uint32_t token = item / spans, h0 = item % spans * per_wave;
        const uint32_t b = token / a.seq, s = token % a.seq;
        const double position = a.positions[token];
        float c[kPairs], sn[kPairs];
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
            const uint32_t p = lane + 64 * e;
            if (p < pairs) {
                float cosine, sine;
                turn(position * a.rates[p], cosine, sine);
                c[e] = cosine * a.magnitude;
                sn[e] = a.inverse ? -sine * a.magnitude : sine * a.magnitude;
            }
        }
        for (uint32_t h = h0; h < min(h0 + per_wave, all); ++h) {
            const Head head = head_of(a, b, s, h);
            float inv = 1.f;
            if constexpr (NORM) {
                float sum = 0.f;
                for (uint32_t d = lane; d < a.dim; d += 64) sum = fmaf(head.x[d], head.x[d], sum);
#pragma unroll
                for (int offset = 32; offset > 0; offset >>= 1) sum += __shfl_xor(sum, offset);
                inv = rsqrtf(sum / float(a.dim) + a.epsilon);
            }
            auto value = [&](uint32_t d) { return NORM ? head.x[d] * inv * head.weight[d] : head.x[d]; };
#pragma unroll
            for (int e = 0; e < kPairs; ++e) {
                const uint32_t p = lane + 64 * e;
                if (p >= pairs) continue;
                const uint32_t da = a.interleaved ? 2 * p : p, db = a.interleaved ? da + 1 : p + pairs;
                const float x = value(da), y = value(db);
                head.out[da] = x * c[e] - y * sn[e];
                head.out[db] = y * c[e] + x * sn[e];
            }
            for (uint32_t d = a.rotary_dim + lane; d < a.dim; d += 64) head.out[d] = value(d);
        }
    }
}

// Lanes per head of rotary_lanes; 0 for rotary_any: parts of a head that are no
// multiple of eight dims.
uint32_t lanes_of(uint32_t dim, uint32_t rotary_dim) {
    if (dim % 8 || rotary_dim % 8) return 0;
    uint32_t lanes = 4;
    while (lanes < dim / 8) lanes *= 2;
    return lanes;
}

struct Split {
    uint32_t per_wave, spans, items, blocks;  // head groups a wave takes, waves per token, waves, blocks
};
// Waves with several groups of heads share their angles, as long as the chip has its
// waves (2048 of them are one for each SIMD twice).
Split split_of(uint32_t tokens, uint32_t heads, uint32_t lanes) {
    const uint32_t groups = lanes ? (heads + 64 / lanes - 1) / (64 / lanes) : heads;
    uint32_t per_wave = 1;
    while (per_wave < 8 && per_wave < groups && uint64_t(tokens) * ((groups + 2 * per_wave - 1) / (2 * per_wave)) >= 2048)
        per_wave *= 2;
    const uint32_t spans = (groups + per_wave - 1) / per_wave, items = tokens * spans;
    const uint32_t blocks = (items + kThreads / 64 - 1) / (kThreads / 64);
    return {per_wave, spans, items, blocks < kMaxBlocks ? blocks : kMaxBlocks};
}

template <bool NORM>
hipError_t launch(hipStream_t stream, const RotaryArgs &a, bool aligned) {
    const uint32_t lanes = aligned ? lanes_of(a.dim, a.rotary_dim) : 0;
    const Split p = split_of(a.batch * a.seq, a.heads + a.heads2, lanes);
    const dim3 grid(p.blocks), block(kThreads);
    switch (lanes) {
        case 0: hipLaunchKernelGGL((rotary_any<NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
        case 4: hipLaunchKernelGGL((rotary_lanes<4, NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
        case 8: hipLaunchKernelGGL((rotary_lanes<8, NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
        case 16: hipLaunchKernelGGL((rotary_lanes<16, NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
        case 32: hipLaunchKernelGGL((rotary_lanes<32, NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
        default: hipLaunchKernelGGL((rotary_lanes<64, NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
    }
    return hipGetLastError();
}

}  // namespace

LaunchShape rotary_shape(uint32_t tokens, uint32_t heads, uint32_t dim, uint32_t rotary_dim, bool norm) {
    const uint32_t lanes = lanes_of(dim, rotary_dim);
    static const char *const names[2][2] = {{"rotary_any", "rotary_lanes"}, {"qk_norm_rotary_any", "qk_norm_rotary_lanes"}};
    return {names[norm][lanes != 0], {split_of(tokens, heads, lanes).blocks, 1, 1}, {kThreads, 1, 1}, 0};
}

hipError_t rotary_f32(hipStream_t stream, const RotaryArgs &a) {
    uintptr_t bits = 0;
    for (const float *p : {a.x, a.x2, a.weight, a.weight2, const_cast<const float *>(a.out),
                           const_cast<const float *>(a.out2)})
        bits |= reinterpret_cast<uintptr_t>(p);
    const bool aligned = (bits & 15u) == 0;
    return a.weight ? launch<true>(stream, a, aligned) : launch<false>(stream, a, aligned);
}

}  // namespace hipk
}  // namespace jade
