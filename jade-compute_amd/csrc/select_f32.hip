// A beam search's selection (beam_select): of every token of every beam, its score
// plus the token's log-probability,
//   score_b + logit_bt - log sum_u exp(logit_bu),
// the `picks` best of a search, best first, ties to the lower beam, then token. A
// finished beam goes on with its `end` token alone and keeps its score.
//
// One pass over the logits. A block takes a chunk of one beam's into registers, and from
// there its maximum, its sum of exponentials and its best tokens, by value and token as
// one 64-bit key: from the least of the four waves' own bounds on every wave has a quarter
// of the picks, so nothing below it is among the best; the few values from there on go to
// LDS and are ranked by counting those above each. A second launch joins the chunks of a
// search in the same way: sums, then the sorted lists' first scores in 64 bits, then the
// entries of those lists whose first one counts. Values that all but tie with their bound
// (equal logits) do not fit the list in LDS: then the best are found one after the other.
//
// 64 searches of 8 beams over 131071 tokens, 16 picks: 57 us for the chunks, 4.7 TB/s,
// bound by vector instructions (chunks of 4096 logits took 73, a chunk loaded ahead 94, 6
// waves a SIMD in fewer registers 76; the greatest bound of a wave that has all of the picks,
// which lets more values through, 62), and 9 for the join. One search of 4 beams over
// 32000: 5 and 6 us; 64 such of 64 picks: 14 and 16 (152 together with one wave's bound and
// every entry looked at); 3 of 16 beams over 50257, 32 picks: 8 and 11 (56).
//
// Beams are compared with one another by their sums of exponentials, so those are summed
// in 64 bits, term by term (adding neighbours in 32 first lost half a part in 2^24 for good where
// one is tiny, and took 1-2% less). A term is off by an ulp of exp2 and two roundings; its
// argument's own rounding is carried along.
#include <cmath>

#include "kernels.hpp"

namespace jade {
namespace hipk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;
constexpr uint32_t kListed = 1024;       // values that a block ranks at once
constexpr uint32_t kMaxBlocks = 1u << 20;
constexpr uint32_t kRawBuffer = 0x00020000;  // buffer descriptor word 3: raw buffer, 32-bit data format
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eRest = 1.92596299112661746887e-8f;  // log2(e) less the float above
constexpr float kLn2 = 0.693147180559945309417f;

// Keys in the order of their values; NaN does not occur.
__device__ inline uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ inline float value_of(uint32_t key) {
    return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ inline uint64_t ordered(double x) {
    const uint64_t b = uint64_t(__double_as_longlong(x));
    return b ^ (b >> 63 ? ~0ull : 1ull << 63);
}
__device__ inline double value_of(uint64_t key) {
    return __longlong_as_double(int64_t(key ^ (key >> 63 ? 1ull << 63 : ~0ull)));
}
// A logit and its token as one key: larger logits first, then lower tokens; no zero is
// below another.
__device__ inline uint64_t key_of(float x, uint32_t token) { return uint64_t(ordered(x + 0.f)) << 32 | ~token; }
constexpr uint32_t kNone = 0x007fffffu;        // ordered(-INFINITY)
constexpr uint64_t kNone64 = 0x000fffffffffffffull;

// A chunk's best tokens, and the maximum and the sum of exp(logit - maximum) of all of them.
struct Space {
    float *value;     // [chunk of all][list]; -inf past the last
    uint32_t *token;
    double *sum;
    float *top;
};
__host__ __device__ inline Space space_of(float *workspace, uint64_t items, uint32_t list) {
    double *const sum = reinterpret_cast<double *>(workspace);
    float *const value = reinterpret_cast<float *>(sum + items);
    uint32_t *const token = reinterpret_cast<uint32_t *>(value + items * list);
    return {value, token, sum, reinterpret_cast<float *>(token + items * list)};
}

// exp(x - top), x <= top and top finite, off by an ulp of exp2 and two roundings: the
// argument's roundings are put back to first order. Nothing of 2^-126 or less counts.
__device__ inline float exp_below(float x, float top) {
    const float d = fmaxf(x - top, -100.f);
    const float lost = __builtin_amdgcn_fmed3f(x - (d + top), -1.f, 1.f);  // x = top + d + lost, but for those
    const float hi = d * kLog2e, lo = fmaf(lost, kLog2e, fmaf(d, kLog2eRest, fmaf(d, kLog2e, -hi)));
    const float e = __builtin_amdgcn_exp2f(hi);
    return fmaf(e, lo * kLn2, e);
}

__device__ inline float wave_max(float x) {
#pragma unroll
    for (int d = 32; d; d /= 2) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}
__device__ inline double wave_sum(double x) {
#pragma unroll
    for (int d = 32; d; d /= 2) x += __shfl_xor(x, d);
    return x;
}
__device__ inline uint64_t wave_max(uint64_t x) {
#pragma unroll
    for (int d = 32; d; d /= 2) {
        const uint64_t y = __shfl_xor(static_cast<unsigned long long>(x), d);
        x = x > y ? x : y;
    }
    return x;
}

// A lower bound of the n-th largest of the wave's 64 keys, n at most 64: its 20 high bits.
__device__ inline uint32_t nth_bound(uint32_t key, uint32_t n) {
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t more = bound | 1u << bit;
        if (uint32_t(__popcll(__ballot(key >= more))) >= n) bound = more;
    }
    return bound;
}

// V: float4s a thread.
template <int V>
__global__ __launch_bounds__(kThreads) void beam_chunks(BeamSelectArgs a, uint32_t chunks, uint32_t items) {
    __shared__ float tops[kWaves];
    __shared__ double sums[kWaves];
    __shared__ uint32_t bounds[kWaves], count;
    __shared__ uint64_t keys[kListed];
    constexpr uint32_t kChunk = 4 * V * kThreads;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid / 64, list = min(a.picks, a.vocab);
    const Space w = space_of(a.workspace, items, list);
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t beam = item / chunks, first = (item - beam * chunks) * kChunk;
        // Nothing of a beam that is finished, or cannot go on, is asked for.
        if (a.finished[beam] > 0.f || !(a.scores[beam] > -INFINITY)) continue;
        // The row's own descriptor: what lies past its end is never read, and vectors need no
        // more than 4-byte alignment.
        const __amdgpu_buffer_rsrc_t row = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<float *>(a.logits + size_t(beam) * a.vocab), 0, int(a.vocab * 4u), int(kRawBuffer));
        auto token_of = [&](int i, int e) { return first + (i * kThreads + tid) * 4 + e; };
        f32x4 x[V];
#pragma unroll
        for (int i = 0; i < V; ++i)
            x[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(row, int(token_of(i, 0) * 4u), 0, 0));
        if (first + kChunk > a.vocab)
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (token_of(i, e) >= a.vocab) x[i][e] = -INFINITY;
        float best[V];  // of four tokens
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = fmaxf(x[i][e], -INFINITY);  // NaN is not chosen
            best[i] = fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3]));
            most = fmaxf(most, best[i]);
        }
        // Every wave has its share of the list from the least of the waves' bounds on; of a
        // row's short end, where waves have nothing, a wave that has all of it counts.
        const bool shared = a.vocab - first >= 4 * kThreads;
        const uint32_t bound = nth_bound(ordered(most + 0.f), shared ? (list + kWaves - 1) / kWaves : list);
        float top = wave_max(most);
        if (lane == 0) {
            tops[wave] = top;
            bounds[wave] = bound;
        }
        if (tid == 0) count = 0;
        __syncthreads();
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const uint32_t least = shared ? min(min(bounds[0], bounds[1]), min(bounds[2], bounds[3]))
                                      : max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3]));
        const float from = value_of(max(least, kNone + 1));
        double sum = 0;
        if (fabsf(top) < INFINITY) {
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += double(exp_below(x[i][e], top));
        } else {  // infinite logits share what there is
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += x[i][e] == top ? 1.0 : 0.0;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (best[i] < from) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (x[i][e] >= from) {
                    const uint32_t at = atomicAdd(&count, 1u);
                    if (at < kListed) keys[at] = key_of(x[i][e], token_of(i, e));
                }
        }
        sum = wave_sum(sum);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        const uint32_t n = count;
        const size_t to = size_t(item) * list;
        if (tid == 0) {
            w.sum[item] = sums[0] + sums[1] + sums[2] + sums[3];
            w.top[item] = top;
        }
        if (n <= kListed) {
            for (uint32_t c = tid; c < n; c += kThreads) {
                const uint64_t mine = keys[c];
                uint32_t rank = 0;
#pragma unroll 8
                for (uint32_t i = 0; i < n; ++i) rank += keys[i] > mine;
                if (rank < list) {
                    w.value[to + rank] = value_of(uint32_t(mine >> 32));
                    w.token[to + rank] = ~uint32_t(mine);
                }
            }
            for (uint32_t i = n + tid; i < list; i += kThreads) w.value[to + i] = -INFINITY;
        } else {
            uint64_t last = ~0ull;
            for (uint32_t r = 0; r < list; ++r) {
                uint64_t best = 0;
#pragma unroll
                for (int i = 0; i < V; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint64_t key = key_of(x[i][e], token_of(i, e));
                        if (key < last && key > best) best = key;
                    }
                best = wave_max(best);
                __syncthreads();
                if (lane == 0) keys[wave] = best;
                __syncthreads();
                last = max(max(keys[0], keys[1]), max(keys[2], keys[3]));
                if (tid == 0) {
                    w.value[to + r] = value_of(uint32_t(last >> 32));
                    w.token[to + r] = ~uint32_t(last);
                }
            }
        }
        __syncthreads();
    }
}

// A candidate's place among the best: by score, then by number (beam * vocab + token).
struct Ranked {
    uint64_t key;
    uint32_t number, unused;
};
__device__ inline bool above(uint64_t key, uint32_t number, uint64_t other, uint32_t others) {
    return key > other || (key == other && number < others);
}

// One block for each search. The chunks' lists are sorted, so a bound of the picks-th largest
// of their first scores bounds what can be among the best, and only lists whose first reaches
// it are looked at further.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void beam_join(BeamSelectArgs a, uint32_t chunks, uint32_t items) {
    constexpr int WAVES = THREADS / 64;
    constexpr uint32_t kLists = 512;  // that are looked at further, at once
    constexpr uint32_t kFew = 256;    // entries that are ranked without another bound
    __shared__ float tops[kMaxBeams], scores[kMaxBeams], ended[kMaxBeams];
    __shared__ double logs[kMaxBeams];
    __shared__ uint64_t counts[2][WAVES];
    __shared__ uint32_t bounds[WAVES], chosen[kLists], count, list_count;
    __shared__ Ranked ranked[kListed];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid / 64, list = min(a.picks, a.vocab);
    const uint32_t b = blockIdx.x, first = b * a.beams, lists = a.beams * chunks;
    const uint32_t spread = lane * WAVES + wave;  // neighbours, often of one beam, go to different waves
    const Space w = space_of(a.workspace, items, list);
    const size_t from_first = size_t(first) * chunks;
    // The first lists' first logits are on their way while the beams' sums are joined.
    const float near = spread < lists ? w.value[(from_first + spread) * list] : 0.f;
    for (uint32_t beam = wave; beam < a.beams; beam += WAVES) {
        const size_t at = size_t(first + beam) * chunks;
        const float score = a.scores[first + beam], end = a.finished[first + beam];
        // The first 64 chunks' maxima and sums together; of a beam that does not go on they
        // are nothing.
        float top = lane < chunks ? w.top[at + lane] : -INFINITY, x = top;
        const double near_sum = lane < chunks ? w.sum[at + lane] : 0.0;
        if (!(end > 0.f) && score > -INFINITY) {
            for (uint32_t i = 64 + lane; i < chunks; i += 64) top = fmaxf(top, w.top[at + i]);
            top = wave_max(top);
            double sum = 0;
            for (uint32_t i = lane; i < chunks; i += 64) {
                if (i >= 64) x = w.top[at + i];
                if (x > -INFINITY) sum += (i >= 64 ? w.sum[at + i] : near_sum) * (x == top ? 1.0 : exp(double(x) - double(top)));
            }
            sum = wave_sum(sum);
            if (lane == 0) logs[beam] = log(sum);
        }
        if (lane == 0) {
            tops[beam] = top;
            scores[beam] = score;
            ended[beam] = end;
        }
    }
    if (tid == 0) count = list_count = 0;
    __syncthreads();
    // The score of entry e, a logit x, of list l; a finished beam has one, in the place of its
    // first.
    auto rate = [&](uint32_t l, uint32_t e, float x) __attribute__((always_inline)) {
        const uint32_t beam = l / chunks;
        const double score = double(scores[beam]);
        if (!(score > -INFINITY)) return kNone64;
        if (ended[beam] > 0.f) return l == beam * chunks && e == 0 && a.end < a.vocab ? ordered(score + 0.0) : kNone64;
        // Infinite logits share what there is.
        const double below = x == tops[beam] ? 0.0 : double(x) - double(tops[beam]);
        if (!(x > -INFINITY) || !(below > -INFINITY)) return kNone64;
        return ordered(below - logs[beam] + score + 0.0);
    };
    auto number_of = [&](uint32_t l, uint32_t e) {
        const uint32_t beam = l / chunks;
        return beam * a.vocab + (ended[beam] > 0.f ? a.end : w.token[(from_first + l) * list + e]);
    };
    // A lower bound of the picks-th largest of the threads' keys: every wave has its share of
    // picks from the least of the waves' bounds on.
    auto bound_of = [&](uint32_t most) {
        const uint32_t bound = nth_bound(most, (a.picks + WAVES - 1) / WAVES);
        if (lane == 0) bounds[wave] = bound;
        __syncthreads();
        uint32_t least = bounds[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) least = min(least, bounds[i]);
        return least;
    };
    // The same to 20 bits, by two bits at a time: where waves differ, some of them with a bad
    // beam's alone.
    auto close_bound_of = [&](uint32_t most) {
        uint32_t bound = 0;
        for (int bit = 30, turn = 0; bit >= 12; bit -= 2, turn ^= 1) {
            const uint32_t one = 1u << bit;
            const uint64_t mine = uint64_t(__popcll(__ballot(most >= (bound | one)))) |
                                  uint64_t(__popcll(__ballot(most >= (bound | 2 * one)))) << 20 |
                                  uint64_t(__popcll(__ballot(most >= (bound | 3 * one)))) << 40;
            if (lane == 0) counts[turn][wave] = mine;
            __syncthreads();
            uint64_t sum = 0;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) sum += counts[turn][i];
            bound += (uint32_t(sum & 0xfffff) >= a.picks) * one + (uint32_t(sum >> 20 & 0xfffff) >= a.picks) * one +
                     (uint32_t(sum >> 40) >= a.picks) * one;
        }
        return bound;
    };
    uint32_t most = spread < lists ? uint32_t(rate(spread, 0, near) >> 32) : 0u;
    for (uint32_t l = spread + THREADS; l < lists; l += THREADS)
        most = max(most, uint32_t(rate(l, 0, w.value[(from_first + l) * list]) >> 32));
    uint32_t from = bound_of(most);
    for (uint32_t l = spread; l < lists; l += THREADS) {
        const uint64_t key = rate(l, 0, l == spread ? near : w.value[(from_first + l) * list]);
        if (key > kNone64 && uint32_t(key >> 32) >= from) {
            const uint32_t at = atomicAdd(&list_count, 1u);
            if (at < kLists) chosen[at] = l;
        }
    }
    __syncthreads();
    // The entries of those lists, all their first ones before their second ones, bounded in
    // the same way where they are many.
    const uint32_t looked = list_count, entries = looked <= kLists ? looked * list : 0;
    auto entry = [&](uint32_t i, uint32_t &l, uint32_t &e) {
        e = i / looked;
        l = chosen[i - e * looked];
        return rate(l, e, w.value[(from_first + l) * list + e]);
    };
    most = 0;
    if (entries > kFew) {
        for (uint32_t i = spread, l, e; i < entries; i += THREADS) most = max(most, uint32_t(entry(i, l, e) >> 32));
        from = max(from, bound_of(most));
    }
    for (int turn = 0;; ++turn) {
        for (uint32_t i = spread, l, e; i < entries; i += THREADS) {
            const uint64_t key = entry(i, l, e);
            if (key > kNone64 && uint32_t(key >> 32) >= from) {
                const uint32_t place = atomicAdd(&count, 1u);
                if (place < kListed) ranked[place] = {key, number_of(l, e), 0};
            }
        }
        __syncthreads();
        if (turn || count <= kFew || entries <= kFew) break;
        from = max(from, close_bound_of(most));
        if (tid == 0) count = 0;
        __syncthreads();
    }
    const uint32_t n = looked <= kLists ? count : kListed + 1;
    const size_t to = size_t(b) * a.picks;
    auto pick = [&](uint32_t rank, uint64_t key, uint32_t number) __attribute__((always_inline)) {
        const uint32_t beam = number / a.vocab, token = number - beam * a.vocab;
        a.parents[to + rank] = float(first + beam);
        a.tokens[to + rank] = float(token);
        a.new_scores[to + rank] = float(value_of(key));
        a.new_finished[to + rank] = token == a.end || ended[beam] > 0.f ? 1.f : 0.f;
    };
    uint32_t got = min(n, a.picks);
    if (n <= kListed) {
        // Four threads for each, of one wave.
        for (uint32_t c = tid / 4; c < n; c += THREADS / 4) {
            const Ranked mine = ranked[c];
            uint32_t rank = 0;
#pragma unroll 4
            for (uint32_t i = tid % 4; i < n; i += 4) rank += above(ranked[i].key, ranked[i].number, mine.key, mine.number);
            rank += __shfl_xor(rank, 1);
            rank += __shfl_xor(rank, 2);
            if (tid % 4 == 0 && rank < a.picks) pick(rank, mine.key, mine.number);
        }
    } else {
        // Scores that all but tie: the best one after the other.
        uint64_t last = ~0ull;
        uint32_t last_number = 0;
        for (got = 0; got < a.picks; ++got) {
            uint64_t best = kNone64;
            uint32_t number = ~0u;
            for (uint32_t c = tid; c < lists * list; c += THREADS) {
                const uint32_t l = c / list, e = c - l * list;
                const uint64_t key = rate(l, e, w.value[from_first * list + c]);
                if (key <= kNone64 || key < best) continue;
                const uint32_t mine = number_of(l, e);
                if (above(last, last_number, key, mine) && above(key, mine, best, number)) {
                    best = key;
                    number = mine;
                }
            }
#pragma unroll
            for (int d = 32; d; d /= 2) {
                const uint64_t key = __shfl_xor(static_cast<unsigned long long>(best), d);
                const uint32_t other = __shfl_xor(number, d);
                if (above(key, other, best, number)) {
                    best = key;
                    number = other;
                }
            }
            __syncthreads();
            if (lane == 0) ranked[wave] = {best, number, 0};
            __syncthreads();
            for (int i = 0; i < WAVES; ++i)
                if (above(ranked[i].key, ranked[i].number, best, number)) {
                    best = ranked[i].key;
                    number = ranked[i].number;
                }
            if (best == kNone64) break;
            last = best;
            last_number = number;
            if (tid == 0) pick(got, best, number);
        }
    }
    for (uint32_t i = got + tid; i < a.picks; i += THREADS) {
        a.parents[to + i] = a.tokens[to + i] = -1.f;
        a.new_scores[to + i] = -INFINITY;
        a.new_finished[to + i] = 0.f;
    }
}

// float4s a thread: the most that leave two blocks a CU and are not more than a row has.
uint32_t words_of(uint32_t batch, uint32_t beams, uint32_t vocab) {
    uint32_t v = 8;
    while (v > 1 && (2 * v * kThreads >= vocab ||
                     uint64_t(batch) * beams * ((vocab + 4 * v * kThreads - 1) / (4 * v * kThreads)) < 512))
        v /= 2;
    return v;
}
uint32_t chunks_of(uint32_t batch, uint32_t beams, uint32_t vocab) {
    const uint32_t chunk = 4 * words_of(batch, beams, vocab) * kThreads;
    return (vocab + chunk - 1) / chunk;
}

template <int V>
void launch_chunks(hipStream_t stream, const BeamSelectArgs &a, uint32_t chunks, uint32_t items) {
    const dim3 grid(items < kMaxBlocks ? items : kMaxBlocks);
    hipLaunchKernelGGL(beam_chunks<V>, grid, dim3(kThreads), 0, stream, a, chunks, items);
}

}  // namespace

LaunchShape beam_select_shape(uint32_t batch, uint32_t beams, uint32_t vocab) {
    const uint32_t items = batch * beams * chunks_of(batch, beams, vocab);  // at most the logits' number
    return {"beam_select", {items < kMaxBlocks ? items : kMaxBlocks, 1, 1}, {kThreads, 1, 1},
            uint32_t(kListed * sizeof(uint64_t) + kWaves * (sizeof(float) + sizeof(double) + sizeof(uint32_t)) + sizeof(uint32_t))};
}

size_t beam_select_workspace_bytes(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t picks) {
    const uint64_t items = uint64_t(batch) * beams * chunks_of(batch, beams, vocab);
    const uint64_t list = picks < vocab ? picks : vocab;
    return items * (sizeof(double) + sizeof(float) + list * (sizeof(float) + sizeof(uint32_t)));
}

hipError_t beam_select_f32(hipStream_t stream, const BeamSelectArgs &a) {
    if (!a.workspace) return hipErrorInvalidValue;
    const uint32_t chunks = chunks_of(a.batch, a.beams, a.vocab), items = a.batch * a.beams * chunks;
    switch (words_of(a.batch, a.beams, a.vocab)) {
        case 8: launch_chunks<8>(stream, a, chunks, items); break;
        case 4: launch_chunks<4>(stream, a, chunks, items); break;
        case 2: launch_chunks<2>(stream, a, chunks, items); break;
        default: launch_chunks<1>(stream, a, chunks, items); break;
    }
    // Sixteen waves where four would take several beams' sums in turn or several lists a
    // thread: 8.8 us against 9.6 for 64 searches of 8 beams, 10 against 18 for 31 of 16, but
    // 7.9 against 6.4 for one of 4 and 38 against 12 for 2000 of 4.
    if (a.beams > 4 || a.beams * chunks > 256)
        hipLaunchKernelGGL(beam_join<1024>, dim3(a.batch), dim3(1024), 0, stream, a, chunks, items);
    else
        hipLaunchKernelGGL(beam_join<kThreads>, dim3(a.batch), dim3(kThreads), 0, stream, a, chunks, items);
    return hipGetLastError();
}

}  // namespace hipk
}  // namespace jade
