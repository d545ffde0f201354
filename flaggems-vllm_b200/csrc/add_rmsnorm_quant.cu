// Residual addition, weighted RMS norm and e4m3 quantisation of hidden states, in one pass over the data.
//
//   z = x + residual (fp32), residual <- z in the tensors' type, r = fp32(1 / sqrt(mean(z^2) + eps)), y = (z * r) * w,
//   scale = max(max |y| of a group, 1e-10) / 448 or the power of two at or above it, x_q = e4m3(y / scale)
//
// Nothing between the sum and the e4m3 byte is rounded to 16 bits.  The mean is formed in 64 bits: squares of fp32 values are exact
// there, so r is the correctly rounded value whatever the order of summation, and with it y, the scales and the bytes are those of the
// definition bit for bit; a power-of-two scale would otherwise move by a factor of two where the last bit of a 32-bit sum carries it
// across.
//
// One CTA per row, the row's sum in registers: thread i holds the 16-byte pieces i, i + blockDim, ..., so every access of a warp is 512
// contiguous bytes and a group of 64 / 128 / 256 values is 8 / 16 / 32 neighbouring lanes.  Bound by HBM: 7 bytes a value.
#include "dsv4_common.cuh"

namespace dsv4 {
namespace {

constexpr float kE4m3Max = 448.0f, kScaleEps = 1e-10f;

struct AddNormParams {
    const uint8_t* x;
    uint8_t* residual;  // may be null: x alone
    const uint8_t* weight;
    uint8_t* out;       // e4m3 [rows, cols], contiguous
    float* scales;
    int64_t x_stride, residual_stride;  // bytes
    int64_t scale_stride_row, scale_stride_group;
    int32_t pieces;       // of 8 values, in a row
    int32_t group_lanes;  // lanes that hold a group; 0: the row is one group
    float eps;
    double inv_cols;
};

struct Bf16 {};
struct Fp16 {};
template <typename T> struct Pair;
template <> struct Pair<Bf16> {
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return make_float2(bf16_lo(u), bf16_hi(u)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
};
template <> struct Pair<Fp16> {
    static __device__ __forceinline__ float2 unpack(uint32_t u) {
        float2 r;
        asm("{.reg .f16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h;}" : "=f"(r.x), "=f"(r.y) : "r"(u));
        return r;
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
        return r;
    }
};

template <typename T>
__device__ __forceinline__ void unpack_piece(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = Pair<T>::unpack(w[i]);
        x[2 * i] = p.x, x[2 * i + 1] = p.y;
    }
}

// Of two values, NaN if either is: a group with a NaN has a NaN scale.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <int PIECES, typename T, bool WEIGHT_F32, int MOST_THREADS>
__global__ void __launch_bounds__(MOST_THREADS) add_rmsnorm_quant_kernel(const Launched<AddNormParams> p, const int pow2) {
    begin_dependent_kernel();
    __shared__ double sums[32];
    __shared__ float maxima[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t row = blockIdx.x;
    const uint8_t* x = p.x + row * p.x_stride;
    uint8_t* residual = p.residual ? p.residual + row * p.residual_stride : nullptr;
    uint4 vx[PIECES], vr[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int at = i * blockDim.x + threadIdx.x;
        vx[i] = vr[i] = make_uint4(0u, 0u, 0u, 0u);
        if (at < p.pieces) {
            vx[i] = ld_inplace16(x + 16 * static_cast<int64_t>(at));
            if (residual) vr[i] = ld_inplace16(residual + 16 * static_cast<int64_t>(at));
        }
    }
    float z[PIECES][8];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int at = i * blockDim.x + threadIdx.x;
        unpack_piece<T>(vx[i], z[i]);
        if (residual) {
            float b[8];
            unpack_piece<T>(vr[i], b);
#pragma unroll
            for (int k = 0; k < 8; ++k) z[i][k] = __fadd_rn(z[i][k], b[k]);
            if (at < p.pieces)
                st_stream16(residual + 16 * static_cast<int64_t>(at), make_uint4(Pair<T>::pack(z[i][0], z[i][1]), Pair<T>::pack(z[i][2], z[i][3]),
                                                                                 Pair<T>::pack(z[i][4], z[i][5]), Pair<T>::pack(z[i][6], z[i][7])));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) sum = fma(static_cast<double>(z[i][k]), static_cast<double>(z[i][k]), sum);
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    sum = lane < warps ? sums[lane] : 0.0;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    const float r = static_cast<float>(1.0 / sqrt(sum * p.inv_cols + static_cast<double>(p.eps)));

    float most[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int at = i * blockDim.x + threadIdx.x;
        float w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = 0.0f;
        if (at < p.pieces) {
            if (WEIGHT_F32) {
                const float4* f = reinterpret_cast<const float4*>(p.weight + 32 * static_cast<int64_t>(at));
                const float4 a = __ldg(f), b = __ldg(f + 1);
                w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
            } else {
                unpack_piece<T>(__ldg(reinterpret_cast<const uint4*>(p.weight + 16 * static_cast<int64_t>(at))), w);
            }
        }
        most[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            z[i][k] = __fmul_rn(__fmul_rn(z[i][k], r), w[k]);
            most[i] = max_or_nan(most[i], fabsf(z[i][k]));
        }
    }
    if (p.group_lanes == 0) {
#pragma unroll
        for (int i = 1; i < PIECES; ++i) most[0] = max_or_nan(most[0], most[i]);
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) most[0] = max_or_nan(most[0], __shfl_xor_sync(0xffffffffu, most[0], m));
        if (lane == 0) maxima[warp] = most[0];
        __syncthreads();
        most[0] = lane < warps ? maxima[lane] : 0.0f;
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) most[0] = max_or_nan(most[0], __shfl_xor_sync(0xffffffffu, most[0], m));
#pragma unroll
        for (int i = 1; i < PIECES; ++i) most[i] = most[0];
    } else {
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            if (m < p.group_lanes) {
#pragma unroll
                for (int i = 0; i < PIECES; ++i) most[i] = max_or_nan(most[i], __shfl_xor_sync(0xffffffffu, most[i], m));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int at = i * blockDim.x + threadIdx.x;
        if (at >= p.pieces) continue;
        float scale = __fdiv_rn(max_or_nan(most[i], kScaleEps), kE4m3Max), q[8];
        if (pow2) {
            // up to the next power of two unless it is one; infinite and NaN scales stay what they are
            if (scale < 0x1p127f) scale = __uint_as_float((__float_as_uint(scale) + 0x7fffffu) & 0x7f800000u);
            const float inverse = __fdiv_rn(1.0f, scale);  // exact, or zero: x / inf
#pragma unroll
            for (int k = 0; k < 8; ++k) q[k] = __fmul_rn(z[i][k], inverse);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) q[k] = __fdiv_rn(z[i][k], scale);
        }
        const uint2 bytes = make_uint2(pack_e4m3x4(q[0], q[1], q[2], q[3]), pack_e4m3x4(q[4], q[5], q[6], q[7]));
        st_global8(p.out + row * (8 * static_cast<int64_t>(p.pieces)) + 8 * static_cast<int64_t>(at), bytes);
        if (p.group_lanes == 0) {
            if (i == 0 && threadIdx.x == 0) p.scales[row * p.scale_stride_row] = scale;
        } else if ((at & (p.group_lanes - 1)) == 0) {
            p.scales[row * p.scale_stride_row + (at / p.group_lanes) * p.scale_stride_group] = scale;
        }
    }
}

template <typename T, bool WEIGHT_F32>
void launch_pieces(int pieces, dim3 grid, int threads, cudaStream_t stream, const AddNormParams& p, int pow2) {
    switch (pieces) {
        case 1: launch_dependent(add_rmsnorm_quant_kernel<1, T, WEIGHT_F32, 1024>, grid, threads, stream, p, pow2); break;
        case 2: launch_dependent(add_rmsnorm_quant_kernel<2, T, WEIGHT_F32, 1024>, grid, threads, stream, p, pow2); break;
        case 3: launch_dependent(add_rmsnorm_quant_kernel<3, T, WEIGHT_F32, 512>, grid, threads, stream, p, pow2); break;
        case 4: launch_dependent(add_rmsnorm_quant_kernel<4, T, WEIGHT_F32, 512>, grid, threads, stream, p, pow2); break;
        case 5: launch_dependent(add_rmsnorm_quant_kernel<5, T, WEIGHT_F32, 512>, grid, threads, stream, p, pow2); break;
        case 6: launch_dependent(add_rmsnorm_quant_kernel<6, T, WEIGHT_F32, 512>, grid, threads, stream, p, pow2); break;
        case 7: launch_dependent(add_rmsnorm_quant_kernel<7, T, WEIGHT_F32, 512>, grid, threads, stream, p, pow2); break;
        default: launch_dependent(add_rmsnorm_quant_kernel<8, T, WEIGHT_F32, 512>, grid, threads, stream, p, pow2); break;
    }
}

}  // namespace

cudaError_t launch_add_rmsnorm_quant(const void* x, int64_t x_stride, void* residual, int64_t residual_stride, const void* weight, void* out,
                                     float* scales, int64_t scale_stride_row, int64_t scale_stride_group, int64_t rows, int64_t cols,
                                     int64_t group_size, float eps, int fp16, int weight_f32, int pow2, cudaStream_t stream) {
    AddNormParams p{};
    p.x = static_cast<const uint8_t*>(x), p.residual = static_cast<uint8_t*>(residual), p.weight = static_cast<const uint8_t*>(weight);
    p.out = static_cast<uint8_t*>(out), p.scales = scales;
    p.x_stride = 2 * x_stride, p.residual_stride = 2 * residual_stride;
    p.scale_stride_row = scale_stride_row, p.scale_stride_group = scale_stride_group;
    p.pieces = static_cast<int32_t>(cols / 8), p.group_lanes = group_size == cols ? 0 : static_cast<int32_t>(group_size / 8);
    p.eps = eps, p.inv_cols = 1.0 / static_cast<double>(cols);
    // Threads for a row: as few as hold it in eight pieces each where many rows share an SM, one piece each where there are few rows.
    const int most = rows <= 148 ? 1 : 8;
    int threads = 128;
    while (threads < 512 && p.pieces > threads * most) threads *= 2;
    if (p.pieces > threads * most && p.pieces <= 2048) threads = 1024;
    const int pieces = (p.pieces + threads - 1) / threads;
    const dim3 grid(static_cast<unsigned>(rows));
    if (fp16) {
        if (weight_f32) launch_pieces<Fp16, true>(pieces, grid, threads, stream, p, pow2);
        else launch_pieces<Fp16, false>(pieces, grid, threads, stream, p, pow2);
    } else {
        if (weight_f32) launch_pieces<Bf16, true>(pieces, grid, threads, stream, p, pow2);
        else launch_pieces<Bf16, false>(pieces, grid, threads, stream, p, pow2);
    }
    count_launch();
    return cudaGetLastError();
}

}  // namespace dsv4
