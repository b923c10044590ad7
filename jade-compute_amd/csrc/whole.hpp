// Whole numbers that travel in FP32 buffers (lengths of sequences): device
// helper shared by the kernels that read them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace jade {
namespace hipk {

// A length: fractions dropped, NaN and what is below 1 taken as 0, what is past
// `most` as `most`. So no buffer's contents lead past the cache.
__device__ inline uint32_t whole_below(float x, uint32_t most) {
    return x >= 1.f ? (x < float(most) ? uint32_t(x) : most) : 0u;
}

}  // namespace hipk
}  // namespace jade
