// Attention over the paged latent cache: queries [tokens, heads, 512] against cached rows of 448 e4m3 values with power-of-two scales and 64
// bf16 values, which are keys and values at once.
//
//   s_j = scale * q . k_j over the keys a token sees, o = sum_j e^(s_j - m) k_j / (sum_j e^(s_j - m) + e^(sink - m)), lse = m + ln sum_j e^(s_j - m)
//
// One warp per (token, head): 16 dimensions a lane, one key after another with a running maximum and sum.
#include "dsv4_common.cuh"
#include "latent_attention.cuh"

namespace dsv4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ue8m0_to_float(uint32_t code) {
    if (code == 0u) return __uint_as_float(0x00400000u);
    if (code == 255u) return __uint_as_float(0x7f800000u);
    return __uint_as_float(code << 23);
}

__global__ void __launch_bounds__(128) latent_attention_kernel(const Launched<LatentAttention> p) {
    begin_dependent_kernel();
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int token = static_cast<int>(row / p.num_heads), head = static_cast<int>(row % p.num_heads);
    if (token >= p.num_tokens) return;
    int request = 0, position = 0, first = 0, low = 0, keys;
    if (p.indices) {
        keys = min(max(__ldg(p.lens + token), 0), p.topk);
    } else {
        while (request < p.num_reqs && __ldg(p.query_start_loc + request + 1) <= token) ++request;
        const int start = request < p.num_reqs ? __ldg(p.query_start_loc + request) : 0;
        if (request == p.num_reqs || token < start) return;
        position = max(__ldg(p.seq_lens + request), 0) - __ldg(p.query_start_loc + request + 1) + token;
        low = p.window > 0 ? max(0, position - p.window + 1) : 0;
        first = min(min(low, p.first), p.capacity);
        keys = max(0, min(position + 1, p.capacity) - low) + first;
    }
    const uint8_t* q = p.q + token * p.q_stride_token + head * p.q_stride_head + 32 * lane;
    float qv[16], acc[16];
    {
        float a[8], b[8];
        unpack8(*reinterpret_cast<const uint4*>(q), a), unpack8(*reinterpret_cast<const uint4*>(q + 16), b);
        for (int i = 0; i < 8; ++i) qv[i] = a[i], qv[8 + i] = b[i];
    }
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < keys; ++j) {
        int64_t block;
        uint32_t in_block;
        if (p.indices) {
            const int slot = __ldg(p.indices + token * p.indices_stride + j);
            if (slot < 0) continue;
            block = fast_div(slot, p.block_mul, p.block_shift);
            in_block = slot - static_cast<uint32_t>(block) * p.block_size;
        } else {
            const int pos = j < first ? j : j - first + low;
            const uint32_t page = fast_div(pos, p.block_mul, p.block_shift);
            in_block = pos - page * p.block_size;
            block = __ldg(p.block_table + request * p.table_stride + page);
        }
        if (block < 0 || block >= p.num_blocks) continue;
        const uint8_t* base = p.k_cache + block * p.block_stride;
        const uint8_t* data = base + static_cast<int64_t>(in_block) * kTokenDataBytes;
        float k[16];
        if (lane < 28) {
            const uint32_t code = base[static_cast<int64_t>(p.block_size) * kTokenDataBytes + static_cast<int64_t>(in_block) * kScaleBytes + (lane >> 2)];
            const float scale = ue8m0_to_float(code);
            const uint4 v = *reinterpret_cast<const uint4*>(data + 16 * lane);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            for (int i = 0; i < 8; ++i) {
                const float2 f = unpack_e4m3x2(static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1))));
                k[2 * i] = f.x * scale, k[2 * i + 1] = f.y * scale;
            }
        } else {
            float a[8], b[8];
            const uint8_t* r = data + kNopeDim + 32 * (lane - 28);
            unpack8(*reinterpret_cast<const uint4*>(r), a), unpack8(*reinterpret_cast<const uint4*>(r + 16), b);
            for (int i = 0; i < 8; ++i) k[i] = a[i], k[8 + i] = b[i];
        }
        float s = 0.0f;
        for (int i = 0; i < 16; ++i) s = fmaf(qv[i], k[i], s);
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= p.scale * kLog2e;
        if (!(s <= m)) {
            const float to = s;
            const float factor = m == -INFINITY ? 0.0f : exp2f(m - to);
            l *= factor;
            for (int i = 0; i < 16; ++i) acc[i] *= factor;
            m = to;
        }
        const float w = m == -INFINITY ? 0.0f : exp2f(s - m);
        l += w;
        for (int i = 0; i < 16; ++i) acc[i] = fmaf(w, k[i], acc[i]);
    }
    if (p.lse && lane == 0)
        p.lse[token * p.lse_stride_token + head * p.lse_stride_head] = l > 0.0f || l != l ? m / kLog2e + logf(l) : -INFINITY;
    float total = l;
    if (p.sink && l > 0.0f) total += exp2f(p.sink[head] * kLog2e - m);
    const float inverse = l == 0.0f ? 0.0f : 1.0f / total;
    uint8_t* out = p.out + token * p.out_stride_token + head * p.out_stride_head + 32 * lane;
    float a[8], b[8];
    for (int i = 0; i < 8; ++i) a[i] = acc[i] * inverse, b[i] = acc[8 + i] * inverse;
    *reinterpret_cast<uint4*>(out) = pack8(a), *reinterpret_cast<uint4*>(out + 16) = pack8(b);
}

}  // namespace

size_t latent_attention_workspace(int64_t num_tokens, int64_t num_heads) { return 0; }

cudaError_t launch_latent_attention(const LatentAttention& p, void* workspace, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(p.num_tokens) * p.num_heads;
    launch_dependent(latent_attention_kernel, static_cast<unsigned>((rows + 3) / 4), 128, stream, p);
    count_launch();
    return cudaGetLastError();
}

}  // namespace dsv4
