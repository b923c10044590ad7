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
// (off by at most 2^-24 of itself), into Taylor series (FP32 angles are off by
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

// Rows that take whole vectors of W floats: LANES lanes (a power of two) share a head,
// a lane with two vectors of it: W pairs, or 2 W dims that are not turned, each vector
// beside its neighbour lane's. A wave keeps one token's angles and goes over `per_wave`
// groups of 64 / LANES heads.
//
// Bound by memory: 4 x 4096 tokens of 32 heads of 128, interleaved, 537 MB in 92.8 us (5.8
// TB/s; 110.9 with a lane's two float4s side by side and ordinary loads and stores).
template <int LANES, int W, bool NORM>
__global__ __launch_bounds__(kThreads) void rotary_lanes(RotaryArgs a, uint32_t per_wave, uint32_t spans,
                                                         uint32_t items) {
    typedef float vec __attribute__((ext_vector_type(W)));
    constexpr int kHalf = W > 1 ? W / 2 : 1;
    const int lane = threadIdx.x & 63;
    const uint32_t unit = lane % LANES, all = a.heads + a.heads2, turned = a.rotary_dim / (2 * W);
    const bool mine = unit < a.dim / (2 * W), turns = unit < turned;
    // Half of the turned dims, or of the others, lies between a lane's two vectors; single
    // floats of an interleaved pair are neighbours.
    const bool near = W == 1 && a.interleaved;
    const uint32_t d0 = turns ? (near ? 2 * unit : W * unit) : a.rotary_dim + W * (unit - turned);
    const uint32_t d1 = turns && near ? d0 + 1 : d0 + (turns ? a.rotary_dim : a.dim - a.rotary_dim) / 2;
    for (uint32_t item = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); item < items;
         item += gridDim.x * (kThreads / 64)) {
        const uint32_t token = item / spans, h0 = item % spans * per_wave * (64 / LANES);
        const uint32_t b = token / a.seq, s = token % a.seq;
        float c[W], sn[W];
        if (turns) {
            const double position = a.positions[token];
#pragma unroll
            for (int e = 0; e < W; ++e) {
                float cosine, sine;
                // The lane's pairs: of halves W unit + e, else half of them in each vector.
                const uint32_t pair = W > 1 && a.interleaved ? kHalf * unit + e % kHalf + e / kHalf * (a.rotary_dim / 4) : W * unit + e;
                turn(position * a.rates[pair], cosine, sine);
                c[e] = cosine * a.magnitude;
                sn[e] = a.inverse ? -sine * a.magnitude : sine * a.magnitude;
            }
        }
        for (uint32_t i = 0; i < per_wave; ++i) {
            const uint32_t h = h0 + i * (64 / LANES) + lane / LANES;
            const bool live = h < all && mine;
            if (!NORM && !live) continue;
            const Head head = head_of(a, b, s, h < all ? h : 0);
            vec x0 = 0.f, x1 = 0.f;
            if (live) {
                x0 = __builtin_nontemporal_load(reinterpret_cast<const vec *>(head.x + d0));
                x1 = __builtin_nontemporal_load(reinterpret_cast<const vec *>(head.x + d1));
            }
            if constexpr (NORM) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < W; ++e) sum = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], sum));
#pragma unroll
                for (int offset = LANES / 2; offset > 0; offset >>= 1) sum += __shfl_xor(sum, offset);
                const float inv = rsqrtf(sum / float(a.dim) + a.epsilon);
                if (!live) continue;
                x0 = x0 * inv * *reinterpret_cast<const vec *>(head.weight + d0);
                x1 = x1 * inv * *reinterpret_cast<const vec *>(head.weight + d1);
            }
            vec y0 = x0, y1 = x1;
            if (turns) {
                if (W > 1 && a.interleaved) {
#pragma unroll
                    for (int e = 0; e < W / 2; ++e) {
                        y0[2 * e] = x0[2 * e] * c[e] - x0[2 * e + 1] * sn[e];
                        y0[2 * e + 1] = x0[2 * e + 1] * c[e] + x0[2 * e] * sn[e];
                        y1[2 * e] = x1[2 * e] * c[W / 2 + e] - x1[2 * e + 1] * sn[W / 2 + e];
                        y1[2 * e + 1] = x1[2 * e + 1] * c[W / 2 + e] + x1[2 * e] * sn[W / 2 + e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        y0[e] = x0[e] * c[e] - x1[e] * sn[e];
                        y1[e] = x1[e] * c[e] + x0[e] * sn[e];
                    }
                }
            }
            __builtin_nontemporal_store(y0, reinterpret_cast<vec *>(head.out + d0));
            __builtin_nontemporal_store(y1, reinterpret_cast<vec *>(head.out + d1));
        }
    }
}

// Odd head dims, and even ones too long for the lanes: one wave a head, pairs and single
// dims in turn.
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

// How rotary_lanes takes a head: the widest vectors of which half the turned dims and half
// the others are whole numbers, and lanes per head; 0 lanes for rotary_any.
struct Lanes {
    uint32_t lanes, width;
};
Lanes lanes_of(uint32_t dim, uint32_t rotary_dim, bool aligned) {
    for (uint32_t width = aligned ? 4 : 1; width; width /= 2) {
        if (dim % (2 * width) || rotary_dim % (2 * width)) continue;
        const uint32_t units = dim / (2 * width);
        return {units <= 8 ? 8u : units <= 16 ? 16u : units <= 32 ? 32u : units <= 64 ? 64u : 0u, width};
    }
    return {0, 1};
}

struct Split {
    uint32_t per_wave, spans, items, blocks;  // head groups a wave takes, waves per token, waves, blocks
};
// Waves with several groups of heads share their angles, as long as the chip has all the
// waves it holds (1531 tokens of 24 heads of 80: 10.0 us where 2048 were enough, 9.2 so).
// The next head loaded ahead of this one's stores: 117.5 -> 115.0 with a norm, but 93 ->
// 94 without and 90 -> 108 for heads of 66 in single floats; not kept.
constexpr uint32_t kLeastWaves = 8192;
Split split_of(uint32_t tokens, uint32_t heads, uint32_t lanes) {
    const uint32_t groups = lanes ? (heads + 64 / lanes - 1) / (64 / lanes) : heads;
    uint32_t per_wave = 1;
    while (per_wave < 8 && per_wave < groups && uint64_t(tokens) * ((groups + 2 * per_wave - 1) / (2 * per_wave)) >= kLeastWaves)
        per_wave *= 2;
    const uint32_t spans = (groups + per_wave - 1) / per_wave, items = tokens * spans;
    const uint32_t blocks = (items + kThreads / 64 - 1) / (kThreads / 64);
    return {per_wave, spans, items, blocks < kMaxBlocks ? blocks : kMaxBlocks};
}

template <int W, bool NORM>
void launch_lanes(hipStream_t stream, const RotaryArgs &a, uint32_t lanes, Split p) {
    const dim3 grid(p.blocks), block(kThreads);
    switch (lanes) {
        case 8: hipLaunchKernelGGL((rotary_lanes<8, W, NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
        case 16: hipLaunchKernelGGL((rotary_lanes<16, W, NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
        case 32: hipLaunchKernelGGL((rotary_lanes<32, W, NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
        default: hipLaunchKernelGGL((rotary_lanes<64, W, NORM>), grid, block, 0, stream, a, p.per_wave, p.spans, p.items); break;
    }
}

template <bool NORM>
hipError_t launch(hipStream_t stream, const RotaryArgs &a, bool aligned) {
    const Lanes l = lanes_of(a.dim, a.rotary_dim, aligned);
    const Split p = split_of(a.batch * a.seq, a.heads + a.heads2, l.lanes);
    if (!l.lanes)
        hipLaunchKernelGGL((rotary_any<NORM>), dim3(p.blocks), dim3(kThreads), 0, stream, a, p.per_wave, p.spans, p.items);
    else if (l.width == 4)
        launch_lanes<4, NORM>(stream, a, l.lanes, p);
    else if (l.width == 2)
        launch_lanes<2, NORM>(stream, a, l.lanes, p);
    else
        launch_lanes<1, NORM>(stream, a, l.lanes, p);
    return hipGetLastError();
}

}  // namespace

LaunchShape rotary_shape(uint32_t tokens, uint32_t heads, uint32_t dim, uint32_t rotary_dim, bool norm) {
    const uint32_t lanes = lanes_of(dim, rotary_dim, true).lanes;
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
