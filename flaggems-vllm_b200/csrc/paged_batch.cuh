// Arguments of the block-table operators, between the C entry points and the kernels.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dsv4 {

constexpr int64_t kMostRequests = 8192;  // of a step: their sums are held in shared memory

struct PagedBatch {
    const int32_t *context_lens, *new_lens;  // [num_reqs]; released: the first alone, with all of a request's tokens
    const uint8_t* finished;                 // released only
    int32_t* block_table;                    // extended; read where it is released from
    int64_t table_stride;
    const int32_t* free_blocks;  // the stack of free blocks, of which *num_free are there,
    int32_t* free_to;            // the same where blocks come back to it
    const int32_t* num_free;
    int32_t *query_start_loc, *seq_lens, *token_to_req, *num_free_out, *num_missing;
    int64_t *position_ids, *slot_mapping;
    int64_t num_tokens;
    int32_t num_reqs, max_blocks, free_capacity;
    uint32_t block_size, block_mul, block_shift;
};

cudaError_t launch_extend_block_tables(const PagedBatch& p, cudaStream_t stream);
cudaError_t launch_release_block_tables(const PagedBatch& p, cudaStream_t stream);

}  // namespace dsv4
