// Arguments of the attention over the paged latent cache, between the C entry points and the kernels.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dsv4 {

struct LatentAttention {
    const uint8_t* q;      // bf16 [num_tokens, num_heads, 512], strides in bytes
    uint8_t* out;          // the same
    float* lse;            // may be null, strides in elements
    const float* sink;     // fp32 [num_heads], may be null
    const uint8_t* k_cache;
    int64_t q_stride_token, q_stride_head, out_stride_token, out_stride_head, lse_stride_token, lse_stride_head;
    int64_t block_stride;  // bytes between cache blocks
    // lists of slots (indices not null), or requests with a block table
    const int32_t* indices;
    int64_t indices_stride;
    const int32_t* lens;
    const int32_t* block_table;
    int64_t table_stride;
    const int32_t* seq_lens;
    const int32_t* query_start_loc;  // [num_reqs + 1]
    float scale;
    int32_t num_tokens, num_heads, topk, num_reqs;
    int32_t window, first;  // window 0: none
    int32_t capacity;       // positions that a row of the block table has pages for
    int32_t num_blocks;
    uint32_t block_size, block_mul, block_shift;
    uint32_t wait_retries;  // of a wait inside the kernel, behind the first try, before it gives up
};

constexpr uint32_t kMostWaitRetries = 1u << 22;  // the default: of up to two microseconds each, some seconds in all

size_t latent_attention_workspace(int64_t num_tokens, int64_t num_heads);
cudaError_t launch_latent_attention(const LatentAttention& p, bool mxfp4, void* workspace, cudaStream_t stream);
cudaError_t read_attention_error(int* value);

}  // namespace dsv4
