// Residual addition, weighted RMS norm and e4m3 quantisation of hidden states, in one pass over the data.
//
//   z = x + residual (fp32), residual <- z in the tensors' type, r = fp32(1 / sqrt(mean(z^2) + eps)), y = (z * r) * w,
//   scale = max(max |y| of a group, 1e-10) / 448 or the power of two at or above it, x_q = e4m3(y / scale)
//
// Nothing between the sum and the e4m3 byte is rounded to 16 bits.  The mean is formed in 64 bits: squares of fp32 values are exact
// there, and their sum is off by less than 2^-48 of it in any order.  So r is the definition's 32-bit value but for rows whose root lies that near to the
// middle of two of them (one row in 2^23), and with it y, the scales and the bytes; a power-of-two scale would otherwise move by a factor of two where the
// last bit of a 32-bit sum carries it across.
//
// As many CTAs as fit take rows in turn, the row's sum in registers: thread i holds the 16-byte pieces i, i + blockDim, ..., so every access of a
// warp is 512 contiguous bytes and a group of 64 / 128 / 256 values is 8 / 16 / 32 neighbouring lanes.  The next row is copied to shared memory
// while this one is worked on (with a CTA for each row instead, 4097 x 7168 took 47.7 us).  Bound by HBM, 7 bytes a value, for many long rows: 4097 x 7168
// bf16 38.3 to 39.0 us (a copy of as many bytes takes 82% of that time), 8192 x 4096 fp16, a scale a row, 44 to 49; the rest is the arithmetic, about 60
// instructions a piece.  One to 148 rows: 2.9 us, the latency of one row's loads, two reductions and stores.
#include <algorithm>

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
    int32_t group_lanes, group_shift;  // lanes that hold a group, and their logarithm; 0 lanes: the row is one group
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
__device__ __forceinline__ void unpack_piece(const uint4& v, float2 (&x)[4]) {
    x[0] = Pair<T>::unpack(v.x), x[1] = Pair<T>::unpack(v.y), x[2] = Pair<T>::unpack(v.z), x[3] = Pair<T>::unpack(v.w);
}

// Two values an instruction, each rounded by itself.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 x, x, y, z; mov.b64 {%0, %1}, x;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Of two values, NaN if either is: a group with a NaN has a NaN scale.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 1 / sqrt(v) rounded to 32 bits: Newton's iteration in 64 from the hardware's approximation (relative error 2^-22, then 2^-43, then below
// 2^-52).  Values beyond what a 32-bit start can hold take the library's functions.
__device__ __forceinline__ float inverse_root(double v) {
    if (!(v > 1e-30 && v < 1e30)) return static_cast<float>(1.0 / sqrt(v));
    double y = static_cast<double>(rsqrtf(static_cast<float>(v)));
    const double h = 0.5 * v;
    y = fma(y, fma(-h * y, y, 0.5), y);
    y = fma(y, fma(-h * y, y, 0.5), y);
    return static_cast<float>(y);
}

// x / d from the correctly rounded reciprocal y of d: the quotient x y corrected once by the remainder (Markstein, 1990).  Off by less than 2^-46 of x / d before its
// one rounding, so its byte is that of the IEEE quotient: a test finds every pair of significands near enough to a border of two bytes to differ, and none does.
// (No step of it underflows for a quotient that is not rounded to a zero byte: the scale is at least 2^-43.)
__device__ __forceinline__ float2 divide(float2 x, float d, float y) {
    const float2 q = mul2(x, both(y));
    return fma2(fma2(both(-d), q, x), both(y), q);
}
__device__ __forceinline__ float scale_of(float most) {
    const float v = max_or_nan(most, kScaleEps), y = 1.0f / kE4m3Max, q = __fmul_rn(v, y);
    return v < INFINITY ? __fmaf_rn(__fmaf_rn(-kE4m3Max, q, v), y, q) : v;
}

__device__ __forceinline__ void copy_ahead(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// EXACT: the row is PIECES pieces of every thread, none of which needs a check.
template <int PIECES, typename T, bool WEIGHT_F32, bool EXACT, int MOST_THREADS, int LEAST_CTAS>
__global__ void __launch_bounds__(MOST_THREADS, LEAST_CTAS)
add_rmsnorm_quant_kernel(const Launched<AddNormParams> p, const int64_t rows, const int pow2, const int two_rows) {
    begin_dependent_kernel();
    // [1 or 2 rows][x, residual][PIECES][threads] of 16 bytes, each thread's own: the next row's copy is under way while this one is worked on
    // (except for rows of which no two fit)
    extern __shared__ __align__(16) uint8_t ahead[];
    __shared__ __align__(16) double sums[2][32];
    __shared__ float maxima[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    if (tid < 16 && (tid & 7) >= warps) sums[tid >> 3][tid & 7] = 0.0;  // (the first barrier lies before they are read)
    const uint32_t pitch = 16 * blockDim.x, mine = static_cast<uint32_t>(__cvta_generic_to_shared(ahead)) + 16 * tid;
    const auto inside = [&](int i) { return EXACT || i * static_cast<int>(blockDim.x) + tid < p.pieces; };
    int64_t row = blockIdx.x;
    const uint8_t* x = p.x + row * p.x_stride + 16 * tid;
    uint8_t* residual = p.residual ? p.residual + row * p.residual_stride + 16 * tid : nullptr;
    uint8_t* out = p.out + row * (8 * static_cast<int64_t>(p.pieces)) + 8 * tid;
    const int64_t x_step = gridDim.x * p.x_stride, residual_step = gridDim.x * p.residual_stride, out_step = gridDim.x * (8 * static_cast<int64_t>(p.pieces));
    const auto ask = [&](const uint8_t* from_x, const uint8_t* from_residual, uint32_t to) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if (!inside(i)) continue;
            copy_ahead(to + i * pitch, from_x + i * pitch);
            if (p.residual) copy_ahead(to + (PIECES + i) * pitch, from_residual + i * pitch);
        }
    };
    const auto arrived = [](uint32_t from) {
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
        return v;
    };
    ask(x, residual, mine);
    asm volatile("cp.async.commit_group;" ::: "memory");
    uint4 vw[PIECES][WEIGHT_F32 ? 2 : 1];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
#pragma unroll
        for (int k = 0; k < (WEIGHT_F32 ? 2 : 1); ++k) {
            vw[i][k] = make_uint4(0u, 0u, 0u, 0u);
            if (inside(i)) vw[i][k] = __ldg(reinterpret_cast<const uint4*>(p.weight + (WEIGHT_F32 ? 2 : 1) * (i * pitch + 16 * tid)) + k);
        }
    }
    for (int turn = 0; row < rows; turn ^= 1) {
        const uint32_t here = mine + (two_rows ? turn * 2 * PIECES * pitch : 0);
        if (two_rows) {
            if (row + gridDim.x < rows) ask(x + x_step, residual + residual_step, mine + (turn ^ 1) * 2 * PIECES * pitch);
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 1;" ::: "memory");
        } else {
            if (row != blockIdx.x) ask(x, residual, mine);
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
        float2 z[PIECES][4];
        double sum[2] = {0.0, 0.0};
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if (!inside(i)) {
#pragma unroll
                for (int k = 0; k < 4; ++k) z[i][k] = both(0.0f);
                continue;
            }
            unpack_piece<T>(arrived(here + i * pitch), z[i]);
            if (p.residual) {
                float2 b[4];
                unpack_piece<T>(arrived(here + (PIECES + i) * pitch), b);
#pragma unroll
                for (int k = 0; k < 4; ++k) z[i][k] = add2(z[i][k], b[k]);
                st_stream16(residual + i * pitch, make_uint4(Pair<T>::pack(z[i][0].x, z[i][0].y), Pair<T>::pack(z[i][1].x, z[i][1].y),
                                                             Pair<T>::pack(z[i][2].x, z[i][2].y), Pair<T>::pack(z[i][3].x, z[i][3].y)));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double a = z[i][k].x, b = z[i][k].y;
                sum[0] = fma(a, a, sum[0]), sum[1] = fma(b, b, sum[1]);
            }
        }
        double total = sum[0] + sum[1];
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) total += __shfl_xor_sync(0xffffffffu, total, m);
        if (lane == 0) sums[turn][warp] = total;
        __syncthreads();
        if (warps <= 8) {
            const double2* parts = reinterpret_cast<const double2*>(sums[turn]);
            const double2 a = parts[0], b = parts[1], c = parts[2], d = parts[3];
            total = ((a.x + a.y) + (b.x + b.y)) + ((c.x + c.y) + (d.x + d.y));
        } else {
            total = lane < warps ? sums[turn][lane] : 0.0;
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) total += __shfl_xor_sync(0xffffffffu, total, m);
        }
        const float r = inverse_root(total * p.inv_cols + static_cast<double>(p.eps));

        float most[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            float2 w[4];
            if constexpr (WEIGHT_F32) {
                const uint4 a = vw[i][0], b = vw[i][1];
                w[0] = make_float2(__uint_as_float(a.x), __uint_as_float(a.y)), w[1] = make_float2(__uint_as_float(a.z), __uint_as_float(a.w));
                w[2] = make_float2(__uint_as_float(b.x), __uint_as_float(b.y)), w[3] = make_float2(__uint_as_float(b.z), __uint_as_float(b.w));
            } else {
                unpack_piece<T>(vw[i][0], w);
            }
            most[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                z[i][k] = mul2(mul2(z[i][k], both(r)), w[k]);
                most[i] = max_or_nan(most[i], max_or_nan(fabsf(z[i][k].x), fabsf(z[i][k].y)));
            }
        }
        if (p.group_lanes == 0) {
#pragma unroll
            for (int i = 1; i < PIECES; ++i) most[0] = max_or_nan(most[0], most[i]);
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) most[0] = max_or_nan(most[0], __shfl_xor_sync(0xffffffffu, most[0], m));
            if (lane == 0) maxima[turn][warp] = most[0];
            __syncthreads();
            most[0] = lane < warps ? maxima[turn][lane] : 0.0f;
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
        float* scales = p.scales + row * p.scale_stride_row;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if (!inside(i)) continue;
            float scale = scale_of(most[i]);
            float2 q[4];
            if (pow2 && scale < 0x1p126f) {
                // up to the next power of two unless it is one, and its exact reciprocal
                const uint32_t bits = (__float_as_uint(scale) + 0x7fffffu) & 0x7f800000u;
                scale = __uint_as_float(bits);
                const float2 inverse = both(__uint_as_float(0x7f000000u - bits));
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = mul2(z[i][k], inverse);
            } else if (scale < INFINITY) {
                const float y = __frcp_rn(scale);
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = divide(z[i][k], scale, y);
            } else {  // infinite: finite values become zero, infinite ones NaN; NaN
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = make_float2(__fdiv_rn(z[i][k].x, scale), __fdiv_rn(z[i][k].y, scale));
            }
            st_global8(out + i * (pitch / 2), make_uint2(pack_e4m3x4(q[0].x, q[0].y, q[1].x, q[1].y), pack_e4m3x4(q[2].x, q[2].y, q[3].x, q[3].y)));
            if (p.group_lanes == 0) {
                if (i == 0 && tid == 0) *scales = scale;
            } else {
                const int at = i * blockDim.x + tid;
                if ((at & (p.group_lanes - 1)) == 0) scales[(at >> p.group_shift) * p.scale_stride_group] = scale;
            }
        }
        row += gridDim.x, x += x_step, residual += residual_step, out += out_step;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int PIECES, typename T, bool WEIGHT_F32, bool EXACT>
cudaError_t launch_rows(int64_t rows, int threads, cudaStream_t stream, const AddNormParams& p, int pow2) {
    // 1024 threads an SM at 64 registers (one or two pieces), 768 at 80 (four), 512 at 128
    constexpr int kMost = PIECES == 1 ? 1024 : PIECES == 2 ? 128 : PIECES == 4 ? 256 : 512, kSmThreads = PIECES <= 2 ? 1024 : PIECES == 4 ? 768 : 512;
    const auto kernel = add_rmsnorm_quant_kernel<PIECES, T, WEIGHT_F32, EXACT, kMost, kSmThreads / kMost>;
    const int row_bytes = 2 * PIECES * threads * 16, two_rows = row_bytes <= 52 * 1024, shared_bytes = (1 + two_rows) * row_bytes;
    // From 48 KiB on, the kernel's own `sums` and `maxima` included, the function has to allow it: the same number each time, the most that any row takes (8 pieces of 512
    // threads), so that a call on another thread with shorter rows does not take it back.
    constexpr int kOwnBytes = 2 * 32 * (sizeof(double) + sizeof(float)), kMostBytes = 2 * 8 * 512 * 16;
    if (shared_bytes + kOwnBytes > 48 * 1024) {
        const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostBytes);
        if (rc != cudaSuccess) return rc;
    }
    // CTAs that fit on an SM, each of which takes rows in turn.
    const int per_sm = std::max(1, std::min({kSmThreads / ((threads + 127) / 128 * 128), 208 * 1024 / (shared_bytes + 2048), 16}));
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(rows, 148LL * per_sm)));
    const cudaError_t rc = launch_dependent_cluster(kernel, grid, dim3(threads), 1, shared_bytes, stream, p, rows, pow2, two_rows);
    if (rc != cudaSuccess) return rc;
    count_launch();
    return cudaGetLastError();
}

template <typename T, bool WEIGHT_F32>
cudaError_t launch_pieces(int pieces, int64_t rows, int threads, cudaStream_t stream, const AddNormParams& p, int pow2) {
    if (pieces == 1) return launch_rows<1, T, WEIGHT_F32, false>(rows, threads, stream, p, pow2);
    if (pieces == 8) return launch_rows<8, T, WEIGHT_F32, false>(rows, threads, stream, p, pow2);
    if (pieces == 2)
        return p.pieces == 2 * threads ? launch_rows<2, T, WEIGHT_F32, true>(rows, threads, stream, p, pow2)
                                       : launch_rows<2, T, WEIGHT_F32, false>(rows, threads, stream, p, pow2);
    return p.pieces == 4 * threads ? launch_rows<4, T, WEIGHT_F32, true>(rows, threads, stream, p, pow2)
                                   : launch_rows<4, T, WEIGHT_F32, false>(rows, threads, stream, p, pow2);
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
    while ((1 << p.group_shift) < p.group_lanes) ++p.group_shift;
    p.eps = eps, p.inv_cols = 1.0 / static_cast<double>(cols);
    // Pieces a thread.  Few rows: one, for the shortest way (148 x 7168: one 3.0 us, four 3.6; 149: 4.5 | 4.2).  Many: more, so that a row's fixed cost, its
    // reductions and barriers, falls on fewer warps (4097 x 7168: one 49 us, four 39, eight 57; 8192 x 2048: one 26.1, two 20.2, four 27.8; 8192 x 1024: one
    // 15.3, two 12.3; 8192 x 768: 14.9 | 12.6; 8192 x 512: 8.7 | 9.9), as far as the registers hold them.
    const auto threads_for = [&](int each) { return ((p.pieces + each - 1) / each + 31) / 32 * 32; };
    const int pieces = p.pieces <= 64 || (rows <= 148 && p.pieces <= 1024) ? 1 : p.pieces <= 256 ? 2 : p.pieces <= 1024 ? 4 : 8;
    const int threads = threads_for(pieces);
    if (fp16) return weight_f32 ? launch_pieces<Fp16, true>(pieces, rows, threads, stream, p, pow2) : launch_pieces<Fp16, false>(pieces, rows, threads, stream, p, pow2);
    return weight_f32 ? launch_pieces<Bf16, true>(pieces, rows, threads, stream, p, pow2) : launch_pieces<Bf16, false>(pieces, rows, threads, stream, p, pow2);
}

}  // namespace dsv4
