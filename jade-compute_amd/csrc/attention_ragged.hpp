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

// The kernel on bf16 parts (attention_ragged_parts.hip), with 32 or 64 rows a block and
// tiles of kPartsTile keys. Needs dim at most 128, 16-byte aligned rows where they are
// whole float4s, and k_row < 2^22.
constexpr uint32_t kPartsTile = 128;
void launch_ragged_parts(hipStream_t stream, const RaggedArgs &args, uint32_t block_rows);
uint32_t ragged_parts_lds_bytes(uint32_t dim, uint32_t block_rows);

}  // namespace hipk
}  // namespace jade
