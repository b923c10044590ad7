// Rows of keys and values appended to a cache: cache row lengths[b] + i takes
// source row picks[b, i], for every head, as long as the picks are whole numbers
// below `rows` and the cache has room; the first pick that is neither ends the
// list. Nothing else of the caches is written.
#include "kernels.hpp"
#include "whole.hpp"

namespace jade {
namespace hipk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr uint32_t kRows = 16;  // cache rows a block writes

__device__ inline bool valid_pick(float p, uint32_t rows) { return p >= 0.f && p < float(rows) && p == truncf(p); }

// Picks of batch b before the first that is not valid, looking at `most` of them,
// for all threads of the block.
__device__ inline uint32_t count_picks(const CacheAppendArgs &a, uint32_t b, uint32_t most) {
    __shared__ uint32_t least;
    if (threadIdx.x == 0) least = most;
    __syncthreads();
    const float *picks = a.picks + size_t(b) * a.picks_count;
    for (uint32_t i = threadIdx.x; i < most; i += kThreads)
        if (!valid_pick(picks[i], a.rows)) {
            atomicMin(&least, i);
            break;
        }
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

template <typename T, bool COUNTED>
__global__ __launch_bounds__(kThreads) void cache_append(CacheAppendArgs a, uint32_t spans, uint32_t items) {
    constexpr uint32_t kWide = sizeof(T) / sizeof(float);
    const uint32_t wide = a.dim / kWide;
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t span = item % spans, rest = item / spans, h = rest % a.kv_heads, b = rest / a.kv_heads;
        const uint32_t first = span * kRows, start = whole_below(a.lengths[b], a.capacity);
        uint32_t count;
        if (COUNTED) {
            count = uint32_t(a.new_lengths[b]) - start;
        } else {
            // The first block of a sequence also writes its new length.
            const bool whole = h == 0 && span == 0;
            const uint32_t most = whole ? a.picks_count : min(a.picks_count, first + kRows);
            count = min(count_picks(a, b, most), a.capacity - start);
            if (whole && threadIdx.x == 0) a.new_lengths[b] = float(start + count);
        }
        if (count <= first) continue;
        const uint32_t n = min(count - first, kRows) * wide;
        const size_t from_row = a.token_major ? size_t(a.kv_heads) * wide : wide;
        const size_t from = a.token_major ? size_t(b) * a.rows * from_row + size_t(h) * wide
                                          : (size_t(b) * a.kv_heads + h) * a.rows * wide;
        const size_t to = (a.token_major ? size_t(b) * a.capacity * from_row + size_t(h) * wide
                                         : (size_t(b) * a.kv_heads + h) * a.capacity * wide) +
                          size_t(start + first) * from_row;
        const float *picks = a.picks + size_t(b) * a.picks_count + first;
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t row = i / wide, d = i % wide;
            const size_t source = from + size_t(picks[row]) * from_row + d, place = to + row * from_row + d;
            reinterpret_cast<T *>(a.k_cache)[place] = reinterpret_cast<const T *>(a.k)[source];
            reinterpret_cast<T *>(a.v_cache)[place] = reinterpret_cast<const T *>(a.v)[source];
        }
    }
}

constexpr uint32_t kMaxBlocks = 1u << 20;
// A block of the one-launch form reads all the picks before its own; past this
// many the counting launch costs less.
constexpr uint32_t kCountedPicks = 16384;

uint32_t spans_of(uint32_t picks) { return (picks + kRows - 1) / kRows; }
uint64_t items_of(uint32_t batch, uint32_t kv_heads, uint32_t picks) {
    return uint64_t(batch) * kv_heads * spans_of(picks);
}

template <typename T>
hipError_t launch(hipStream_t stream, const CacheAppendArgs &a) {
    const uint32_t items = uint32_t(items_of(a.batch, a.kv_heads, a.picks_count));
    const dim3 grid(items < kMaxBlocks ? items : kMaxBlocks), block(kThreads);
    if (a.picks_count > kCountedPicks) {
        hipLaunchKernelGGL(cache_count, dim3(a.batch), block, 0, stream, a);
        hipLaunchKernelGGL((cache_append<T, true>), grid, block, 0, stream, a, spans_of(a.picks_count), items);
    } else {
        hipLaunchKernelGGL((cache_append<T, false>), grid, block, 0, stream, a, spans_of(a.picks_count), items);
    }
    return hipGetLastError();
}

}  // namespace

LaunchShape cache_append_shape(uint32_t batch, uint32_t kv_heads, uint32_t picks) {
    const uint64_t items = items_of(batch, kv_heads, picks);
    if (items > 0xffffffffull) return {nullptr, {0, 0, 0}, {0, 0, 0}, 0};
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
