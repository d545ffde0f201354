// Block tables and slots of a step, made on the GPU from the lengths of its requests, and the way back of a finished request's blocks.
//
// extend_block_tables: request r has c_r tokens in the cache and gets n_r new ones.  With b tokens a block and w entries a row of the block table it holds
// h_r = min(ceil(c_r / b), w) blocks and takes t_r = min(ceil((c_r + n_r) / b), w) - h_r more: the i-th block that is taken, counted over all requests in
// order, is free[top - 1 - i].  So with T_r = sum of t before r and S_r = sum of n before r every table entry and every token is a formula of its own:
//   entry h_r + k of row r is free[top - 1 - T_r - k], token S_r + j has position c_r + j, whose slot follows from that entry, or from the table where k < 0.
// A CTA holds the sums of all requests in shared memory and finds a token's (an entry's) request by bisection.  What is read and written is a few bytes a
// token, so the time is that of the dependent loads (lengths, then entries) and of the launch.  One launch does all: up to eight CTAs, a cluster, each with
// the sums of its own (eight bytes a request to read), so that none waits for another; the cluster's barrier only keeps the results that may
// replace their arguments (num_free, seq_lens) back until every CTA has read those.
//
// release_block_tables: the entries e_0, e_1, ... of the finished requests' rows, in order, go to free[top + count - 1 - i]: what undoes the taking.  Entries
// that are negative (blocks that were missing) are left out, so a warp a request counts them first; the CTAs of the cluster tell each other.
#include "dsv4_common.cuh"
#include "paged_batch.cuh"

namespace dsv4 {
namespace {

constexpr int kMostThreads = 1024, kMostCluster = 8;
// Tokens (and finished requests' entries) that one CTA takes before another joins it.
constexpr int64_t kTokensPerCta = 2048;

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
// Writes to the same place of the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ void store_cluster(const int32_t* at, uint32_t rank, int32_t v) {
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.b32 [a], %2;\n\t}" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(at))),
                 "r"(rank), "r"(v)
                 : "memory");
}

__device__ __forceinline__ int32_t saturated(int64_t v) { return v > 0x7fffffffLL ? 0x7fffffff : static_cast<int32_t>(v); }
// Blocks of `tokens` tokens, at most a row of the table.
__device__ __forceinline__ int32_t blocks_of(const PagedBatch& p, int32_t tokens) {
    const uint32_t whole = fast_div(static_cast<uint32_t>(tokens), p.block_mul, p.block_shift);
    return min(static_cast<int32_t>(whole + (whole * p.block_size != static_cast<uint32_t>(tokens) ? 1u : 0u)), p.max_blocks);
}

// Exclusive sum of a pair over the CTA's threads, and the total in `total`.  All threads take part; `sums` has an entry per warp.
__device__ __forceinline__ longlong2 sum_before(longlong2 mine, longlong2* sums, longlong2& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    longlong2 up_to = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, up_to.x, d), y = __shfl_up_sync(0xffffffffu, up_to.y, d);
        if (lane >= d) up_to.x += x, up_to.y += y;
    }
    if (lane == 31) sums[warp] = up_to;
    __syncthreads();
    longlong2 before = make_longlong2(up_to.x - mine.x, up_to.y - mine.y);
    total = make_longlong2(0, 0);
    for (int w = 0; w < warps; ++w) {
        const longlong2 s = sums[w];
        if (w < warp) before.x += s.x, before.y += s.y;
        total.x += s.x, total.y += s.y;
    }
    return before;
}

// The first of `count` non-decreasing numbers that is greater than `v`; `count` if there is none.
template <typename T>
__device__ __forceinline__ int first_above(const T* ends, int count, int64_t v) {
    int low = 0, high = count;
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (ends[mid] > v) high = mid;
        else low = mid + 1;
    }
    return low;
}

__global__ void __launch_bounds__(kMostThreads) extend_block_tables_kernel(const Launched<PagedBatch> p) {
    begin_dependent_kernel();
    extern __shared__ __align__(16) uint8_t shared[];
    __shared__ longlong2 sums[kMostThreads / 32];
    int64_t* block_ends = reinterpret_cast<int64_t*>(shared);  // per request: blocks taken up to its own,
    int32_t* token_ends = reinterpret_cast<int32_t*>(block_ends + p.num_reqs);  // new tokens up to its own,
    int32_t* contexts = token_ends + p.num_reqs;                                // tokens in the cache
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const int tid = threadIdx.x, reqs = p.num_reqs;

    const int64_t top = min(max(*p.num_free, 0), p.free_capacity);
    const int each = (reqs + blockDim.x - 1) / blockDim.x, begin = min(tid * each, reqs), end = min(begin + each, reqs);
    longlong2 mine = make_longlong2(0, 0), total;
    for (int r = begin; r < end; ++r) {
        const int32_t c = max(p.context_lens[r], 0), n = max(__ldg(p.new_lens + r), 0);
        contexts[r] = c;
        mine.x += blocks_of(p, saturated(static_cast<int64_t>(c) + n)) - blocks_of(p, c);
        mine.y += n;
        block_ends[r] = mine.x;
    }
    longlong2 before = sum_before(mine, sums, total);
    cluster_arrive();  // num_free and the contexts have been read
    for (int r = begin; r < end; ++r) {
        before.y += max(__ldg(p.new_lens + r), 0);
        block_ends[r] += before.x;
        token_ends[r] = saturated(before.y);
    }
    __syncthreads();

    const int64_t first = static_cast<int64_t>(rank) * blockDim.x + tid, stride = static_cast<int64_t>(ctas) * blockDim.x;
    const auto taken = [&](int64_t i) { return i < top ? __ldg(p.free_blocks + (top - 1 - i)) : -1; };
    const auto blocks_before = [&](int r) { return r > 0 ? block_ends[r - 1] : 0; };
    for (int64_t t = first; t < p.num_tokens; t += stride) {
        const int r = first_above(token_ends, reqs, t);
        int64_t position = 0, slot = -1;
        if (r < reqs) {
            const int32_t c = contexts[r];
            position = c + (t - (r > 0 ? token_ends[r - 1] : 0));
            if (position <= 0x7fffffffLL) {
                const uint32_t page = fast_div(static_cast<uint32_t>(position), p.block_mul, p.block_shift);
                const int32_t held = blocks_of(p, c);
                if (page < static_cast<uint32_t>(p.max_blocks)) {
                    const int64_t block = static_cast<int32_t>(page) < held ? p.block_table[r * p.table_stride + page] : taken(blocks_before(r) + page - held);
                    if (block >= 0) slot = block * p.block_size + (static_cast<uint32_t>(position) - page * p.block_size);
                }
            }
        }
        p.position_ids[t] = position;
        p.slot_mapping[t] = slot;
        p.token_to_req[t] = r < reqs ? r : 0;
    }
    for (int64_t i = first; i < total.x; i += stride) {
        const int r = first_above(block_ends, reqs, i);
        p.block_table[r * p.table_stride + blocks_of(p, contexts[r]) + (i - blocks_before(r))] = taken(i);
    }
    cluster_wait();
    for (int64_t r = first; r < reqs; r += stride) {
        p.query_start_loc[r + 1] = token_ends[r];
        p.seq_lens[r] = saturated(static_cast<int64_t>(contexts[r]) + max(__ldg(p.new_lens + r), 0));
    }
    if (first == 0) {
        const int64_t out = total.x < top ? total.x : top;
        p.query_start_loc[0] = 0;
        *p.num_free_out = static_cast<int32_t>(top - out);
        *p.num_missing = saturated(total.x - out);
    }
}

// f(entry number, entry) for the entries of a request's row that this lane has, eight loads at a time; the warp's lanes have neighbouring ones.
constexpr int kAtOnce = 8;
template <typename F>
__device__ __forceinline__ void for_entries(const int32_t* row, int count, int lane, F&& f) {
    for (int k = 0; k < count; k += 32 * kAtOnce) {
        int32_t e[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) e[i] = k + 32 * i + lane < count ? __ldg(row + k + 32 * i + lane) : -1;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (k + 32 * i < count) f(e[i]);
    }
}

__global__ void __launch_bounds__(kMostThreads) release_block_tables_kernel(const Launched<PagedBatch> p) {
    begin_dependent_kernel();
    extern __shared__ __align__(16) uint8_t shared[];
    __shared__ longlong2 sums[kMostThreads / 32];
    int64_t* befores = reinterpret_cast<int64_t*>(shared);             // per request: blocks of the finished ones in front of it,
    int32_t* counts = reinterpret_cast<int32_t*>(befores + p.num_reqs);  // its own, if it is finished
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5, reqs = p.num_reqs;
    const int first = rank * warps + (tid >> 5), stride = ctas * warps;
    const int64_t top = min(max(*p.num_free, 0), p.free_capacity);
    cluster_arrive();
    cluster_wait();  // every CTA of the cluster runs, and its shared memory may be written
    const auto entries_of = [&](int r) { return __ldg(p.finished + r) != 0 ? blocks_of(p, max(__ldg(p.context_lens + r), 0)) : 0; };
    for (int r = first; r < reqs; r += stride) {
        int count = 0;
        for_entries(p.block_table + r * p.table_stride, entries_of(r), lane, [&](int32_t e) { count += e >= 0; });
        count = __reduce_add_sync(0xffffffffu, count);
        if (lane < ctas) store_cluster(counts + r, lane, count);
    }
    cluster_arrive();  // (num_free has been read as well)
    cluster_wait();
    const int each = (reqs + blockDim.x - 1) / blockDim.x, begin = min(tid * each, reqs), end = min(begin + each, reqs);
    longlong2 mine = make_longlong2(0, 0), total;
    for (int r = begin; r < end; ++r) mine.x += counts[r];
    longlong2 before = sum_before(mine, sums, total);
    for (int r = begin; r < end; ++r) befores[r] = before.x, before.x += counts[r];
    __syncthreads();
    for (int r = first; r < reqs; r += stride) {
        int64_t to = top + total.x - 1 - befores[r];
        for_entries(p.block_table + r * p.table_stride, entries_of(r), lane, [&](int32_t e) {
            const uint32_t live = __ballot_sync(0xffffffffu, e >= 0);
            const int64_t at = to - __popc(live & ((1u << lane) - 1u));
            if (e >= 0 && at < p.free_capacity) p.free_to[at] = e;
            to -= __popc(live);
        });
    }
    if (rank == 0 && tid == 0) *p.num_free_out = static_cast<int32_t>(min(top + static_cast<int64_t>(total.x), static_cast<int64_t>(p.free_capacity)));
}

cudaError_t launch(void (*kernel)(const Launched<PagedBatch>), const PagedBatch& p, int64_t items, int64_t per_cta, size_t shared_bytes, cudaStream_t stream) {
    unsigned cluster = 1;
    while (cluster < kMostCluster && items > cluster * per_cta) cluster *= 2;
    const int64_t most = items > p.num_reqs ? items : p.num_reqs;
    const unsigned threads = most <= 128 ? 128 : most <= 512 ? 512 : kMostThreads;
    if (shared_bytes > 40 * 1024) {
        const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared_bytes));
        if (rc != cudaSuccess) return rc;
    }
    const cudaError_t rc = launch_dependent_cluster(kernel, dim3(cluster), dim3(threads), cluster, shared_bytes, stream, p);
    if (rc != cudaSuccess) return rc;
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_extend_block_tables(const PagedBatch& p, cudaStream_t stream) {
    return launch(extend_block_tables_kernel, p, p.num_tokens, kTokensPerCta, 16 * static_cast<size_t>(p.num_reqs), stream);
}

cudaError_t launch_release_block_tables(const PagedBatch& p, cudaStream_t stream) {
    // a warp a request
    return launch(release_block_tables_kernel, p, 32 * static_cast<int64_t>(p.num_reqs), kMostThreads, 12 * static_cast<size_t>(p.num_reqs), stream);
}

}  // namespace dsv4
