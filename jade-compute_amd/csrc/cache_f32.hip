// Rows of keys and values appended to a cache: cache row lengths[b] + i takes
// source row picks[b, i], for every head, as long as the picks are whole numbers
// below `rows` and the cache has room; the first pick that is neither ends the
// list. Nothing else of the caches is written.
//
// A copy, bound by memory: K and V in one launch, whole float4s where rows allow it,
// loads and stores past the L2 (nothing reads them again here). A block copies 2 float4s a
// thread of each tensor: 4 sequences x 4096 rows x 8 heads x 128 in 49 us, 5.5 TB/s; a few
// rows take what a launch takes (3.5 us).
#include "kernels.hpp"
#include "whole.hpp"

namespace jade {
namespace hipk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr uint32_t kBlockWords = 2 * kThreads;  // elements (float4s, or floats) of each tensor that a block copies

__device__ inline bool valid_pick(float p, uint32_t rows) { return p >= 0.f && p < float(rows) && p == truncf(p); }

// Picks of batch b before the first that is not valid, looking at `most` of them,
// for all threads of the block.
__device__ inline uint32_t count_picks(const CacheAppendArgs &a, uint32_t b, uint32_t most) {
    __shared__ uint32_t least;
    if (threadIdx.x == 0) least = most;
    __syncthreads();
    const float *picks = a.picks + size_t(b) * a.picks_count;
    uint32_t bad = most;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < most; i += kThreads)
        if (!valid_pick(picks[i], a.rows)) bad = min(bad, i);
    if (bad < most) atomicMin(&least, bad);
    __syncthreads();
    const uint32_t got = least;
    __syncthreads();
    return got;
}

// Long lists: every sequence's new length by a launch of its own, so that the
// copying blocks need not look at all the picks before theirs.
__global__ __launch_bounds__(kThreads) void cache_count(CacheAppendArgs a) {
    const uint32_t start = whole_below(a.lengths[blockIdx.x], a.capacity);
    const uint32_t count = min(count_picks(a, blockIdx.x, a.picks_count), a.capacity - start);
    if (threadIdx.x == 0) a.new_lengths[blockIdx.x] = float(start + count);
}

// Rows of `wide` elements; tokens of all heads are one row where they lie together
// (`heads` is 1 then). A block takes `span` rows of one head.
template <typename T, bool COUNTED>
__global__ __launch_bounds__(kThreads) void cache_append(CacheAppendArgs a, uint32_t heads, uint32_t wide, uint32_t span,
                                                         uint32_t spans, uint32_t items) {
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t at = item % spans, rest = item / spans, h = rest % heads, b = rest / heads;
        const uint32_t first = at * span, start = whole_below(a.lengths[b], a.capacity);
        uint32_t count;
        if (COUNTED) {
            count = uint32_t(a.new_lengths[b]) - start;
        } else {
            // The first block of a sequence also writes its new length.
            const bool whole = h == 0 && at == 0;
            const uint32_t most = whole ? a.picks_count : min(a.picks_count, first + span);
            count = min(count_picks(a, b, most), a.capacity - start);
            if (whole && threadIdx.x == 0) a.new_lengths[b] = float(start + count);
        }
        if (count <= first) continue;
        const uint32_t n = min(count - first, span) * wide;
        const size_t from = size_t(rest) * a.rows * wide, to = (size_t(rest) * a.capacity + start + first) * wide;
        const float *picks = a.picks + size_t(b) * a.picks_count + first;
#pragma unroll 2
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t row = i / wide;
            const size_t source = from + size_t(picks[row]) * wide + (i - row * wide);
            const T k = __builtin_nontemporal_load(reinterpret_cast<const T *>(a.k) + source);
            const T v = __builtin_nontemporal_load(reinterpret_cast<const T *>(a.v) + source);
            __builtin_nontemporal_store(k, reinterpret_cast<T *>(a.k_cache) + to + i);
            __builtin_nontemporal_store(v, reinterpret_cast<T *>(a.v_cache) + to + i);
        }
    }
}

constexpr uint32_t kMaxBlocks = 1u << 20;
// A block of the one-launch form reads all the picks before its own, some of them again
// from the L2; the counting launch costs 2 us. 8 heads of 128: 4096 picks 17.1 us counted,
// 15.5 in one launch; 8192 28.3 and 28.2; 16384 52 and 57; 65536 200 and 366.
constexpr uint32_t kCountedPicks = 8192;

struct Split {
    uint32_t heads, wide, span, spans;
    uint64_t items;
};
Split split_of(uint32_t batch, uint32_t kv_heads, uint32_t picks, uint32_t dim, bool token_major, bool vec) {
    Split s;
    s.heads = token_major ? 1 : kv_heads;
    s.wide = (token_major ? kv_heads * dim : dim) / (vec ? 4 : 1);
    s.span = s.wide < kBlockWords ? kBlockWords / s.wide : 1;
    s.spans = (picks + s.span - 1) / s.span;
    s.items = uint64_t(batch) * s.heads * s.spans;
    return s;
}

template <typename T>
hipError_t launch(hipStream_t stream, const CacheAppendArgs &a) {
    const Split s = split_of(a.batch, a.kv_heads, a.picks_count, a.dim, a.token_major, sizeof(T) == 16);
    const uint32_t items = uint32_t(s.items);
    const dim3 grid(items < kMaxBlocks ? items : kMaxBlocks), block(kThreads);
    if (a.picks_count > kCountedPicks) {
        hipLaunchKernelGGL(cache_count, dim3(a.batch), block, 0, stream, a);
        hipLaunchKernelGGL((cache_append<T, true>), grid, block, 0, stream, a, s.heads, s.wide, s.span, s.spans, items);
    } else {
        hipLaunchKernelGGL((cache_append<T, false>), grid, block, 0, stream, a, s.heads, s.wide, s.span, s.spans, items);
    }
    return hipGetLastError();
}

}  // namespace

LaunchShape cache_append_shape(uint32_t batch, uint32_t kv_heads, uint32_t picks, uint32_t dim, bool token_major) {
    const uint64_t items = split_of(batch, kv_heads, picks, dim, token_major, dim % 4 == 0).items;
    if (items > 0xfffffffeull - kMaxBlocks) return {nullptr, {0, 0, 0}, {0, 0, 0}, 0};
    return {picks > kCountedPicks ? "cache_append_counted" : "cache_append",
            {uint32_t(items < kMaxBlocks ? items : kMaxBlocks), 1, 1}, {kThreads, 1, 1}, uint32_t(sizeof(uint32_t))};
}

hipError_t cache_append_f32(hipStream_t stream, const CacheAppendArgs &a) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                           reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache);
    return a.dim % 4 == 0 && (bits & 15u) == 0 ? launch<f32x4>(stream, a) : launch<float>(stream, a);
}

}  // namespace hipk
}  // namespace jade
