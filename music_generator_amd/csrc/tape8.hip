// The 8-bit activation tape (format: tape8.h): packing, unpacking, and the product of a gradient with the SoftRectifier
// derivative recovered from a kept output.  The reference keeps its activations in float32 (tf.GradientTape,
// trainer/models.py:118); the backward convolution that reads this form is bbwd_kernel in bwgrad.hip.
//
// All three are bound by HBM: 3.03 bytes a value for bf16, 5.03 for float32 and 5.03 for the product.  Four lanes share a
// block and a lane moves eight values (16 bytes of bf16, 8 of codes), so the block's maximum is two exchanges inside a
// group of four lanes and every load and store of a wave covers consecutive bytes.  Measured: product with the derivative of
// 2 x 128 x 24000 x 128 values 4.5 TB/s (879 us, 1415 with the packing; a large copy reaches 4.75).
#include "tape8.h"
#include "../../include/mgx.h"

namespace {

constexpr int kBlock = 256;
constexpr long kMaxGrid = 4096;

inline unsigned grid_for(long items) {
    long g = (items + kBlock - 1) / kBlock;
    if (g > kMaxGrid) g = kMaxGrid;
    return (unsigned)g;
}

inline bool misaligned(const void* p) { return ((uintptr_t)p & 15u) != 0; }

// values 8 i .. 8 i + 7 as float32; those past the end are zeros
template <bool F32>
__device__ __forceinline__ void load8(const void* __restrict__ x, long i, long n, float* v) {
    if (8 * i + 8 <= n) {
        if (F32) {
            const f32x4 a = ((const f32x4*)x)[2 * i], b = ((const f32x4*)x)[2 * i + 1];
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[k] = a[k]; v[4 + k] = b[k]; }
        } else {
            const u32x4 a = ((const u32x4*)x)[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[2 * k] = bf_lo(a[k]); v[2 * k + 1] = bf_hi(a[k]); }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const long j = 8 * i + k;
            v[k] = j < n ? (F32 ? ((const float*)x)[j] : (float)((const bf16_t*)x)[j]) : 0.f;
        }
    }
}

template <bool F32>
__device__ __forceinline__ void store8(void* __restrict__ y, long i, long n, const float* v) {
    if (8 * i + 8 <= n) {
        if (F32) {
            ((f32x4*)y)[2 * i] = (f32x4){v[0], v[1], v[2], v[3]};
            ((f32x4*)y)[2 * i + 1] = (f32x4){v[4], v[5], v[6], v[7]};
        } else {
            ((u32x4*)y)[i] = (u32x4){bf_pack(v[0], v[1]), bf_pack(v[2], v[3]), bf_pack(v[4], v[5]), bf_pack(v[6], v[7])};
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const long j = 8 * i + k;
            if (j < n) {
                if (F32) ((float*)y)[j] = v[k];
                else ((bf16_t*)y)[j] = (bf16_t)v[k];
            }
        }
    }
}

// n8: eight-value pieces of whole blocks (the last block's missing values count as zeros and get codes too)
template <bool F32>
__global__ __launch_bounds__(kBlock) void tape8_pack_kernel(const void* __restrict__ x, u32x2* __restrict__ codes,
                                                            unsigned char* __restrict__ exps, long n8, long n) {
    for (long i = (long)blockIdx.x * kBlock + threadIdx.x; i < n8; i += (long)gridDim.x * kBlock) {
        float v[8];
        load8<F32>(x, i, n, v);
        unsigned m = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const unsigned b = __builtin_bit_cast(unsigned, v[k]) & 0x7fffffffu;
            m = m > b ? m : b;
        }
        const unsigned e = tape8_exponent(tape8_quad_max(m));       // n8 is a multiple of 4: the group of four is whole
        const float inv = tape8_inverse(e);
        codes[i] = (u32x2){tape8_code4(v, inv), tape8_code4(v + 4, inv)};
        if ((threadIdx.x & 3) == 0) exps[i >> 2] = (unsigned char)e;
    }
}

template <bool F32>
__global__ __launch_bounds__(kBlock) void tape8_unpack_kernel(const u32x2* __restrict__ codes,
                                                              const unsigned char* __restrict__ exps, void* __restrict__ y,
                                                              long n8, long n) {
    for (long i = (long)blockIdx.x * kBlock + threadIdx.x; i < n8; i += (long)gridDim.x * kBlock) {
        const u32x2 c = codes[i];
        const float step = tape8_step(exps[i >> 2]), off = -127.5f * step;
        float v[8];
        tape8_value4(c[0], step, off, v);
        tape8_value4(c[1], step, off, v + 4);
        store8<F32>(y, i, n, v);
    }
}

// out = a f'(y), y the kept output of tanh(v) + v / alpha
template <bool AF32>
__global__ __launch_bounds__(kBlock) void mul_dact_tape8_kernel(const void* __restrict__ a, const u32x2* __restrict__ codes,
                                                                const unsigned char* __restrict__ exps,
                                                                void* __restrict__ out, long n8, long n, float inv_alpha) {
    const float k1 = 1.0f + inv_alpha;
    for (long i = (long)blockIdx.x * kBlock + threadIdx.x; i < n8; i += (long)gridDim.x * kBlock) {
        const u32x2 c = codes[i];
        const float step = tape8_step(exps[i >> 2]), off = -127.5f * step;
        float v[8], av[8];
        load8<AF32>(a, i, n, av);
        tape8_value4(c[0], step, off, v);
        tape8_value4(c[1], step, off, v + 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = av[k] * tape8_dact(v[k], inv_alpha, k1);
        store8<false>(out, i, n, v);
    }
}

}  // namespace

extern "C" int64_t mgx_tape8_blocks(int64_t n) { return n > 0 ? (n + 31) / 32 : 0; }

extern "C" int mgx_tape8_pack(const void* x, int x_is_f32, void* codes, void* exps, int64_t n, void* stream) {
    if (n < 0) return MGX_ERR_ARG;
    if (n == 0) return MGX_OK;
    if (!x || !codes || !exps || misaligned(x) || misaligned(codes)) return MGX_ERR_ARG;
    const long n8 = mgx_tape8_blocks(n) * 4;
    const dim3 grid(grid_for(n8));
    if (x_is_f32)
        hipLaunchKernelGGL(tape8_pack_kernel<true>, grid, dim3(kBlock), 0, (hipStream_t)stream, x, (u32x2*)codes,
                           (unsigned char*)exps, n8, (long)n);
    else
        hipLaunchKernelGGL(tape8_pack_kernel<false>, grid, dim3(kBlock), 0, (hipStream_t)stream, x, (u32x2*)codes,
                           (unsigned char*)exps, n8, (long)n);
    return mgx_launch_status();
}

extern "C" int mgx_tape8_unpack(const void* codes, const void* exps, void* y, int y_is_f32, int64_t n, void* stream) {
    if (n < 0) return MGX_ERR_ARG;
    if (n == 0) return MGX_OK;
    if (!y || !codes || !exps || misaligned(y) || misaligned(codes)) return MGX_ERR_ARG;
    const long n8 = (n + 7) / 8;
    const dim3 grid(grid_for(n8));
    if (y_is_f32)
        hipLaunchKernelGGL(tape8_unpack_kernel<true>, grid, dim3(kBlock), 0, (hipStream_t)stream, (const u32x2*)codes,
                           (const unsigned char*)exps, y, n8, (long)n);
    else
        hipLaunchKernelGGL(tape8_unpack_kernel<false>, grid, dim3(kBlock), 0, (hipStream_t)stream, (const u32x2*)codes,
                           (const unsigned char*)exps, y, n8, (long)n);
    return mgx_launch_status();
}

extern "C" int mgx_mul_dact_tape8(const void* a, int a_is_f32, const void* codes, const void* exps, float act_alpha,
                                  void* out, int64_t n, void* stream) {
    if (n < 0 || !(act_alpha > 0.f)) return MGX_ERR_ARG;
    if (n == 0) return MGX_OK;
    if (!a || !out || !codes || !exps || misaligned(a) || misaligned(out) || misaligned(codes)) return MGX_ERR_ARG;
    const long n8 = (n + 7) / 8;
    const dim3 grid(grid_for(n8));
    if (a_is_f32)
        hipLaunchKernelGGL(mul_dact_tape8_kernel<true>, grid, dim3(kBlock), 0, (hipStream_t)stream, a, (const u32x2*)codes,
                           (const unsigned char*)exps, out, n8, (long)n, 1.0f / act_alpha);
    else
        hipLaunchKernelGGL(mul_dact_tape8_kernel<false>, grid, dim3(kBlock), 0, (hipStream_t)stream, a, (const u32x2*)codes,
                           (const unsigned char*)exps, out, n8, (long)n, 1.0f / act_alpha);
    return mgx_launch_status();
}
