// Host interface of the ragged attention kernels (attention_ragged.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace jade {
namespace hipk {

// Strides in elements. Rows of q and out are [batch, head, query], of k and v
// [batch, kv head, key], of the drafted kd and vd [batch, kv head, node].
struct RaggedArgs {
    const float *q, *k, *v, *lengths;
    const float *kd, *vd, *parents;  // a tree's drafted keys and values, else null (nodes 0)
    float *out, *partial;
    size_t q_batch, q_head, k_batch, k_head, d_batch, d_head;
    uint32_t q_row, k_row;  // k_row also between drafted rows
    uint32_t batch, kv_heads, group, queries, keys, nodes, dim;
    uint32_t row_blocks, runs;
    float qscale;  // scale * log2(e)
};

}  // namespace hipk
}  // namespace jade
