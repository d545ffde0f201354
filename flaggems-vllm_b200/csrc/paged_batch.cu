// Block tables and slots of a step, made on the GPU from the lengths of its requests, and the way back of a finished request's blocks.
//
// extend_block_tables: request r has c_r tokens in the cache and gets n_r new ones.  With b tokens a block and w entries a row of the block table it holds
// h_r = min(ceil(c_r / b), w) blocks and takes t_r = min(ceil((c_r + n_r) / b), w) - h_r more: the i-th block that is taken, counted over all requests in
// order, is free[top - 1 - i].  So with T_r = sum of t before r and S_r = sum of n before r every table entry and every token is a formula of its own:
//   entry h_r + k of row r is free[top - 1 - T_r - k], token S_r + j has position c_r + j, whose slot follows from that entry, or from the table where k < 0.
// Every CTA makes the sums of all requests for itself (eight bytes a request to read), holds them in shared memory and finds a token's (an entry's) request
// by bisection, so that none waits for another.  What is read and written is a few bytes a token: the time is that of the dependent loads (lengths, then
// entries) and of the launch.  Where a result stands in the place of an argument (num_free, seq_lens), the CTAs are one cluster, whose barrier keeps those two
// back until every CTA has read them, and a cluster has eight at most; otherwise there is a CTA for every 1024 tokens, rounded up to a power of two, up to the number of SMs.
//
// release_block_tables: the entries e_0, e_1, ... of the finished requests' rows, in order, go to free[top + count - 1 - i]: what undoes the taking.  Entries
// that are negative (blocks that were missing) are left out.  The rows' entries are one list, which the warps of a cluster share out evenly: each counts
// its part, the counts go to all CTAs, and each writes behind those in front of it.
//
// GPU time of a call, one behind another in a graph: extend, 1 request 2.4 to 2.6 us, 61 3.3 to 3.5 us, 1021 with 65 thousand new tokens 5.3 to 5.5 us; with its state in place 2.5 to 2.9,
// 3.2 to 3.8 and 14 us (eight CTAs instead of 64).  Release, 61 requests 5.2 to 5.5 us, half of 1021 with 259 thousand entries 17.2 us, bound by the instructions of eight SMs (a search
// for every entry, and a vote for every 32 where none is missing: 25 us; a warp a request 24.8 us, and more where one is long).
#include "dsv4_common.cuh"
#include "paged_batch.cuh"

namespace dsv4 {
namespace {

constexpr int kMostThreads = 1024, kMostCluster = 8, kMostCtas = 148;
constexpr int kBytesPerRequest = 12;  // of the shared memory of extend_block_tables_kernel; the other kernel has 4

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

// Sum over the CTA's threads in front of this one, and the total in `total`.  All threads take part; `sums` has an entry per warp.
template <typename T>
__device__ __forceinline__ T sum_before(T mine, T* sums, T& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    T up_to = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const T x = __shfl_up_sync(0xffffffffu, up_to, d);
        if (lane >= d) up_to += x;
    }
    if (lane == 31) sums[warp] = up_to;
    __syncthreads();
    // every warp sums up the warps for itself
    T of_warps = lane < warps ? sums[lane] : T(0);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const T x = __shfl_up_sync(0xffffffffu, of_warps, d);
        if (lane >= d) of_warps += x;
    }
    total = __shfl_sync(0xffffffffu, of_warps, 31);
    const T in_front = __shfl_sync(0xffffffffu, of_warps, warp > 0 ? warp - 1 : 0);
    return up_to - mine + (warp > 0 ? in_front : T(0));
}

// The first of the non-decreasing numbers ends[low .. high - 1] that is greater than `v`; `high` if there is none.
__device__ __forceinline__ int first_above(const int32_t* ends, int low, int high, int32_t v) {
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
    __shared__ int64_t token_sums[kMostThreads / 32];
    __shared__ int32_t block_sums[kMostThreads / 32];
    int32_t* block_ends = reinterpret_cast<int32_t*>(shared);  // per request: blocks taken up to its own,
    int32_t* token_ends = block_ends + p.num_reqs;             // new tokens up to its own,
    int32_t* contexts = token_ends + p.num_reqs;               // tokens in the cache
    const int tid = threadIdx.x, reqs = p.num_reqs;

    const int32_t top = min(max(*p.num_free, 0), p.free_capacity);
    const int each = (reqs + blockDim.x - 1) / blockDim.x, begin = min(tid * each, reqs), end = min(begin + each, reqs);
    int64_t tokens = 0, all_tokens;
    int32_t blocks = 0, all_blocks;
    for (int r = begin; r < end; ++r) {
        const int32_t c = max(p.context_lens[r], 0), n = max(__ldg(p.new_lens + r), 0);
        contexts[r] = c;
        blocks += blocks_of(p, saturated(static_cast<int64_t>(c) + n)) - blocks_of(p, c);
        tokens += n;
        block_ends[r] = blocks;
    }
    const int32_t blocks_before = sum_before(blocks, block_sums, all_blocks);
    int64_t sum = sum_before(tokens, token_sums, all_tokens);
    cluster_arrive();  // num_free and the contexts have been read
    for (int r = begin; r < end; ++r) {
        sum += max(__ldg(p.new_lens + r), 0);
        block_ends[r] += blocks_before;
        token_ends[r] = saturated(sum);
    }
    __syncthreads();

    const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + tid, stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    const auto taken = [&](int32_t i) { return i < top ? __ldg(p.free_blocks + (top - 1 - i)) : -1; };
    const auto start_of = [&](const int32_t* ends, int r) { return r > 0 ? ends[r - 1] : 0; };
    for (int64_t t = first; t < p.num_tokens; t += stride) {
        const int r = first_above(token_ends, 0, reqs, static_cast<int32_t>(t));
        int64_t position = 0, slot = -1;
        if (r < reqs) {
            const int32_t c = contexts[r];
            position = c + (t - start_of(token_ends, r));
            if (position <= 0x7fffffffLL) {
                const uint32_t page = fast_div(static_cast<uint32_t>(position), p.block_mul, p.block_shift);
                const int32_t held = blocks_of(p, c), before = start_of(block_ends, r);
                // Not behind those that the request has now: lengths end at 2^31 - 1, and with a block of as many tokens position 2^31 - 1 is on a page that is not counted.
                if (page < static_cast<uint32_t>(held + block_ends[r] - before)) {
                    const int64_t block = static_cast<int32_t>(page) < held ? p.block_table[r * p.table_stride + page] : taken(before + static_cast<int32_t>(page) - held);
                    if (block >= 0) slot = block * p.block_size + (static_cast<uint32_t>(position) - page * p.block_size);
                }
            }
        }
        p.position_ids[t] = position;
        p.slot_mapping[t] = slot;
        p.token_to_req[t] = r < reqs ? r : 0;
    }
    for (int64_t i = first; i < all_blocks; i += stride) {
        const int32_t at = static_cast<int32_t>(i);
        const int r = first_above(block_ends, 0, reqs, at);
        p.block_table[r * p.table_stride + blocks_of(p, contexts[r]) + (at - start_of(block_ends, r))] = taken(at);
    }
    cluster_wait();
    for (int64_t r = first; r < reqs; r += stride) {
        p.query_start_loc[r + 1] = token_ends[r];
        p.seq_lens[r] = saturated(static_cast<int64_t>(contexts[r]) + max(__ldg(p.new_lens + r), 0));
    }
    if (first == 0) {
        const int32_t out = min(all_blocks, top);
        p.query_start_loc[0] = 0;
        *p.num_free_out = top - out;
        *p.num_missing = all_blocks - out;
    }
}

constexpr int kAtOnce = 8;  // loads of a lane

__global__ void __launch_bounds__(kMostThreads) release_block_tables_kernel(const Launched<PagedBatch> p) {
    begin_dependent_kernel();
    extern __shared__ __align__(16) uint8_t shared[];
    __shared__ int32_t sums[kMostThreads / 32];
    __shared__ int32_t counts[kMostCluster * kMostThreads / 32];  // per warp of the cluster: blocks that it has
    int32_t* ends = reinterpret_cast<int32_t*>(shared);           // per request: entries of the finished ones up to its own
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5, reqs = p.num_reqs;
    const int all = ctas * warps, own = rank * warps + (tid >> 5);
    const int32_t top = min(max(*p.num_free, 0), p.free_capacity);
    cluster_arrive();
    const int each = (reqs + blockDim.x - 1) / blockDim.x, begin = min(tid * each, reqs), end = min(begin + each, reqs);
    int32_t mine = 0, total;
    for (int r = begin; r < end; ++r) {
        const int32_t tokens = max(__ldg(p.context_lens + r), 0);
        mine += __ldg(p.finished + r) != 0 ? blocks_of(p, tokens) : 0;
        ends[r] = mine;
    }
    const int32_t before = sum_before(mine, sums, total);
    for (int r = begin; r < end; ++r) ends[r] += before;
    __syncthreads();
    // this warp's part of the list, and the requests that it lies in
    const int32_t share = static_cast<int32_t>((static_cast<uint32_t>(total) + all - 1) / all);
    const int32_t from = static_cast<int32_t>(min(static_cast<int64_t>(share) * own, static_cast<int64_t>(total))), to = from + min(share, total - from);
    const int low = first_above(ends, 0, reqs, from), high = to > from ? first_above(ends, low, reqs, to - 1) : low;
    // The entries i, i + 1, ... of it, as far as they exist.  32 of them are mostly of one row; where they are not, every lane searches for its own.
    const auto load = [&](int32_t i, int32_t (&e)[kAtOnce]) {
        const int left = min(to - i, 32 * kAtOnce);
        int r = first_above(ends, low, high, i);
        const auto row_of = [&](int of) { return p.block_table + of * p.table_stride + (i - (of > 0 ? ends[of - 1] : 0)); };
        const int32_t* row = left > 0 ? row_of(r) : p.block_table;
        int end = left > 0 ? ends[r] - i : 0;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int at = 32 * k + lane, behind = min(32 * k + 32, left);
            e[k] = -1;
            if (behind <= end) {
                if (at < left) e[k] = __ldg(row + at);
            } else {
                if (at < left) e[k] = __ldg(row_of(first_above(ends, r, high, i + at)) + at);
                if (behind < left) r = first_above(ends, r, high, i + behind), row = row_of(r), end = ends[r] - i;
            }
        }
    };
    int32_t e[kAtOnce];  // the part's first entries are kept until they are written
    int32_t count = 0;
    for (int32_t i = to > from ? from + (to - 1 - from) / (32 * kAtOnce) * (32 * kAtOnce) : from; i >= from; i -= 32 * kAtOnce) {
        load(i, e);
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) count += e[k] >= 0;
    }
    count = __reduce_add_sync(0xffffffffu, count);
    cluster_wait();  // every CTA of the cluster runs, so that its shared memory may be written, and has read num_free
    if (lane < ctas) store_cluster(counts + own, lane, count);
    cluster_arrive();
    cluster_wait();
    int32_t in_front = 0, blocks = 0;
    for (int w = lane; w < all; w += 32) blocks += counts[w], in_front += w < own ? counts[w] : 0;
    blocks = __reduce_add_sync(0xffffffffu, blocks), in_front = __reduce_add_sync(0xffffffffu, in_front);
    int64_t at = static_cast<int64_t>(top) + blocks - 1 - in_front;
    const bool plain = count == to - from && at < p.free_capacity;  // no entry is left out, and none has no place
    for (int32_t done = 0; done < to - from; done += 32 * kAtOnce) {  // (from + done may pass 2^31 - 1 behind the last round, `done` cannot)
        const int32_t i = from + done;
        if (done > 0) load(i, e);
        if (plain) {
            int32_t* place = p.free_to + (at - done - lane);
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k)
                if (32 * k + lane < to - i) place[-32 * k] = e[k];
            continue;
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const uint32_t live = __ballot_sync(0xffffffffu, e[k] >= 0);
            const int64_t place = at - __popc(live & ((1u << lane) - 1u));
            if (e[k] >= 0 && place < p.free_capacity) p.free_to[place] = e[k];
            at -= __popc(live);
        }
    }
    if (rank == 0 && tid == 0) *p.num_free_out = static_cast<int32_t>(min(static_cast<int64_t>(top) + blocks, static_cast<int64_t>(p.free_capacity)));
}

cudaError_t launch(void (*kernel)(const Launched<PagedBatch>), const PagedBatch& p, int64_t items, unsigned ctas, bool cluster, size_t shared_bytes,
                   cudaStream_t stream) {
    const unsigned threads = items <= 128 ? 128 : items <= 512 ? 512 : kMostThreads;
    if (shared_bytes > 40 * 1024) {
        // The same number each time, the most that any call takes, so that a call on another thread with fewer requests does not take it back.
        const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytesPerRequest * kMostRequests);
        if (rc != cudaSuccess) return rc;
    }
    const cudaError_t rc = launch_dependent_cluster(kernel, dim3(ctas), dim3(threads), cluster ? ctas : 1, shared_bytes, stream, p);
    if (rc != cudaSuccess) return rc;
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_extend_block_tables(const PagedBatch& p, cudaStream_t stream) {
    const bool in_place = p.num_free_out == p.num_free || p.seq_lens == p.context_lens;
    const int64_t most = in_place ? kMostCluster : kMostCtas;
    unsigned ctas = 1;
    while (ctas < most && p.num_tokens > ctas * static_cast<int64_t>(kMostThreads)) ctas *= 2;
    if (ctas > most) ctas = static_cast<unsigned>(most);
    return launch(extend_block_tables_kernel, p, p.num_tokens > p.num_reqs ? p.num_tokens : p.num_reqs, ctas, in_place, kBytesPerRequest * static_cast<size_t>(p.num_reqs), stream);
}

cudaError_t launch_release_block_tables(const PagedBatch& p, cudaStream_t stream) {
    // How many entries there are is known on the GPU alone: a CTA for 16 requests.  With 1 | 2 | 4 | 8 CTAs: 1 request, 16 entries 3.7 | 4.0 | 4.3 | 4.2 us, 16 requests, 176 entries
    // 4.5 | 4.9 | 4.8 | 4.8, 61 requests, 1019 entries 4.9 | 5.3 | 5.5 | 5.1, and 7393 entries 6.5 | 6.0 | 5.7 | 5.3, 256 requests, 2952 entries 5.8 in all four, 1021 requests, 259 thousand
    // entries 102 | 54 | 30 | 17.  Few requests with long rows pay for the rule: 16 with 65536 entries 17.5 | 11.1 | 7.4 | 5.4.
    unsigned ctas = 1;
    while (ctas < kMostCluster && p.num_reqs > ctas * 16) ctas *= 2;
    return launch(release_block_tables_kernel, p, kMostThreads, ctas, true, 4 * static_cast<size_t>(p.num_reqs), stream);
}

}  // namespace dsv4
