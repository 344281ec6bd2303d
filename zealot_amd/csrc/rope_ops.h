// rope_ops.h -- arguments of the norm + rotary pass (rope_ops.hip), shared with
// the KV cache, which calls it with its own slots and positions.
#pragma once

#include "zk_common.h"

namespace zk {

struct RopeArgs {
    const void *q, *k, *v;                 // [T, heads, D] rows, strides in elements (0: packed)
    int64_t q_stride, k_stride, v_stride;  // (v: append only)
    zk_dtype dtype;                        // of q, k, v, the weights, q_out and k_out
    int64_t num_tokens;
    int num_heads, num_kv_heads, head_dim;
    const void *q_weight, *k_weight;  // [D] or null: no norm
    float eps;
    const int32_t *positions;  // [T]
    const float *rope;         // [max_positions][rot_dim]: cosines, then sines
    int64_t max_positions;
    int rot_dim, interleaved;
    void *q_out, *k_out;  // k_out: without pools only
    int64_t q_out_stride, k_out_stride;
    // the KV write (pools null: none)
    void *k_pool, *v_pool;
    zk_dtype cache_dtype;
    const int64_t *slots;  // [T]
    int block_size;
    int64_t num_blocks, num_slots;
    const float *k_scales, *v_scales;
    const int32_t *token_row;
    int lanes;      // of a head in the vector kernel
    float inv_dim;  // 1 / head_dim
};
int qk_norm_rope(const RopeArgs &a, hipStream_t s);
// Its checks of arguments alone.  by_cache: slots, positions, scales and
// token_row are the cache's and not yet known.
int check_qk_norm_rope(const RopeArgs &a, bool by_cache);

}  // namespace zk
