// Softmax cross entropy of a Dense head with many classes, without keeping the logits (beside mgx_softmax_xent, which
// takes them as a tensor: the reference's Dense(9, softmax) + categorical_crossentropy, trainer/evaluacion.py:97, 160).
//     z = x W + b (n x v)     lse_i = log sum_j exp(z_ij)     loss_i = lse_i - z_i,label(i)
//     dz_ij = dloss_i (exp(z_ij - lse_i) - [j = label(i)])    dx = dz W^T    dW = x^T dz    db_j = sum_i dz_ij
// x is n x e (float32 or bf16), W e x v and b v (float32, the Keras layout).  The logits exist in registers (accumulator
// tiles) only: the forward reduces each tile to a maximum and a sum per row, the backward computes them again, turns them into
// dz and feeds dz to the two gradient products.
//
// Arithmetic: few rows in float32.  The products of many rows run on v_mfma_f32_32x32x16_f16 with float32 accumulation, at
// float32 quality.  A float32
// operand is the sum of two fp16 planes, hi = fp16(s a) and lo = fp16(s a - hi) with s a power of two that brings a row of x (each
// its own, so that no row's digits depend on another's), or all of W, below 2^14 in magnitude: 22 significant bits, and 2^-25 of
// 2^14 absolute where a value is small.  The
// product keeps hi hi + hi lo + lo hi (the dropped lo lo is 2^-24 of it).  A bf16 operand is exact in one plane.  This is
// three (two) of 2.5 PFLOP/s instead of one of the 157 TFLOP/s of the float32 matrix instructions.
// Logits, maxima, sums, lse and all gradient sums are float32.  Biases are in units of log 2 and log2(e) is in the factor that
// takes the powers of two out: an exponential is one fma, one difference and one v_exp_f32.  (Accumulators that start at the bias
// times both powers save the difference, but that product leaves float32 where the operands are small or the bias is a mask.)
//
// Four forms.  What each is bound by, and forward + backward times (us; n x e x v):
//   few rows (up to 4, up to 16 of a small W): launches and HBM (W read twice, dW written), float32 on the vector ALU.
//     1 x 128 x 4097 15 + 17, 4 x 128 x 65536 15 + 42.
//   a block of rows (up to 64, 128 of a large W): HBM up to 32 rows (a kernel each for the logits, dx and dW, 4.4 to 4.9 TB/s at 32 x
//     1000 x 65536; a large copy reaches 4.75), the float32 matrix instructions beyond (64 x 1000 x 65536 94 + 260).
//   e <= 128: the matrix pipe, streamed, dz never stored.  24000 x 128 x 65536 bf16: 780 + 2490 (the three products 0.72, 1.11
//     and 1.35 ms, 1.1 to 1.2 PFLOP/s of fp16 products; a library product of 8192^3 reaches 1.22).  The form below takes 1450 +
//     5920 for it, and 1725 + 7320 against 1090 + 3910 for float32 features (products at 1.1 to 1.23); at 3000 x 128 x 8192 bf16
//     41 + 100 against 42 + 92.
//   e > 128: the matrix pipe, tiled products with dz in planes of 128 MB a piece.  1501 x 1000 x 10001 float32: 132 + 346, of which
//     the four products (0.93 PFLOP/s) take 390; bf16 106 + 254.
// Up to 64 features the streamed kernels have a form of 64 (24000 x 32 x 65536 bf16: 440 + 1340 against 680 + 2110 us).
//
// A row whose label lies outside [0, v) has no loss: loss 0, lse 0, gradient 0 and nothing of its features is read into
// a product (they may hold anything).  A class masked with a bias of -inf or the lowest float has a probability of 0, and its column
// of W is not used either; one class at least is not masked.
#include "bf16.h"
#include "../../include/mgx.h"

namespace {

typedef _Float16 f16_t;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16 mfma_f16(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ unsigned f16_pack(float lo, float hi) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){lo, hi}, f16x2));
}

__device__ __forceinline__ unsigned lds_byte(const unsigned char* p) {
    return (unsigned)(size_t)(__attribute__((address_space(3))) const void*)p;
}

// One LDS-DMA instruction: lane l moves 16 (4) bytes from byte `off` of the uniform address `base` to LDS byte dst + 16 l (4 l),
// dst uniform.  Complete when the issuing wave has waited for vmcnt.
__device__ __forceinline__ void lds_dma16(const void* base, int off, unsigned dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void lds_dma4(const void* base, int off, unsigned dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory");
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kLowest = -3.402823466e38f;
// Where the results of the dW products go when the contraction is not split: the gradients themselves (slabs otherwise).
struct XentOut {
    float *dw, *db;               // of the piece's first class
    long v, cnt;                  // classes of W, valid classes of the piece
    int e, accumulate, direct;
};

constexpr float kDz = 16384.f;                     // planes of probabilities hold 2^14 p
constexpr int kMaxParts = 512;

inline int64_t up(int64_t a, int64_t m) { return (a + m - 1) / m * m; }

// ---------------------------------------------------------------- powers of two
// Largest finite magnitudes as float32 bits: of every labelled row of x (rmax), and one partial per workgroup of the unmasked classes of
// W, of the labelled rows' dloss, and of their product with the row's largest (as the sum of both exponents, 1 more: 0 is
// none); what is unlabelled or masked may hold anything.  A thread takes 4 features of 4 classes of W (WVEC, rows of whole 16-byte
// pieces) or 16 features of one; 2^lsh lanes walk a row of x, in pieces of 16 bytes where rows consist of them (VEC).
__device__ __forceinline__ bool masked(float b) { return b <= kLowest; }

template <bool XF32, bool VEC, bool WVEC>
__global__ __launch_bounds__(256) void xent_max_kernel(const float* __restrict__ w, const float* __restrict__ b,
                                                       const void* __restrict__ x, long n, int e, const int* __restrict__ labels,
                                                       long v, int lsh, const float* __restrict__ dl, unsigned* __restrict__ part,
                                                       unsigned* __restrict__ rmax) {
    __shared__ unsigned red[3][4];
    const long t = (long)blockIdx.x * 256 + threadIdx.x, stride = (long)gridDim.x * 256;
    unsigned m[3] = {0u, 0u, 0u};
    auto take = [](unsigned& a, unsigned b) {
        b &= 0x7fffffffu;
        if (b < 0x7f800000u && b > a) a = b;
    };
    constexpr int CL = WVEC ? 4 : 1, FE = 16 / CL;
    const long groups = v / CL, items = groups * ((e + FE - 1) / FE);
    for (long i = t; i < items; i += stride) {
        const long k0 = i / groups * FE, c = (i - i / groups * groups) * CL;
        u32x4 q[4];                                          // all loads in flight
        float bv[CL];
        if constexpr (WVEC) {
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = *(const u32x4*)(w + (k0 + j < e ? k0 + j : e - 1) * v + c);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) q[j >> 2][j & 3] = __builtin_bit_cast(unsigned, w[(k0 + j < e ? k0 + j : e - 1) * v + c]);
        }
#pragma unroll
        for (int k = 0; k < CL; ++k) bv[k] = b ? b[c + k] : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (!masked(bv[WVEC ? k : 0]))
#pragma unroll
                for (int j = 0; j < 4; ++j) take(m[0], q[j][k]);
    }
    constexpr int PER = VEC ? (XF32 ? 4 : 8) : 1;
    const int lanes = 1 << lsh, cols = e / PER;
    for (long row = t >> lsh; row < n; row += stride >> lsh) {
        const int lab = labels[row];
        if (lab < 0 || lab >= v) continue;
        unsigned rm = 0u;
        for (int c = threadIdx.x & (lanes - 1); c < cols; c += 4 * lanes) {
            if constexpr (VEC) {
                u32x4 q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    q[j] = c + j * lanes < cols ? ((const u32x4*)x)[row * cols + c + j * lanes] : (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        take(rm, XF32 ? q[j][k] : q[j][k] & 0xffff0000u);
                        if (!XF32) take(rm, q[j][k] << 16);
                    }
            } else {
                unsigned q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const long at = row * e + c + j * lanes;
                    q[j] = c + j * lanes >= cols ? 0u : XF32 ? ((const unsigned*)x)[at] : (unsigned)((const unsigned short*)x)[at] << 16;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) take(rm, q[j]);
            }
        }
        for (int off = lanes >> 1; off > 0; off >>= 1) {
            const unsigned o = (unsigned)__shfl_xor((int)rm, off, 64);
            rm = rm > o ? rm : o;
        }
        if ((threadIdx.x & (lanes - 1)) == 0) {
            rmax[row] = rm;
            if (dl) {
                unsigned d = 0u;
                take(d, __builtin_bit_cast(unsigned, dl[row]));
                m[2] = m[2] > d ? m[2] : d;
                const unsigned both = d && rm ? (d >> 23) + (rm >> 23) + 1u : 0u;
                m[1] = m[1] > both ? m[1] : both;
            }
        }
    }
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const unsigned o = (unsigned)__shfl_xor((int)m[k], off, 64);
            m[k] = m[k] > o ? m[k] : o;
        }
        if (lane == 0) red[k][wv] = m[k];
    }
    __syncthreads();
    if (threadIdx.x < 3) {
        unsigned a = 0u;
        for (int k = 0; k < 4; ++k) a = a > red[threadIdx.x][k] ? a : red[threadIdx.x][k];
        part[threadIdx.x * kMaxParts + blockIdx.x] = a;
    }
}

// Exponent that brings magnitudes up to the float32 with these bits below 2^14 (max < 2^(field - 126)).
__device__ __forceinline__ int exponent_of(unsigned maxbits) { return maxbits == 0u ? 0 : 140 - (int)(maxbits >> 23); }

// A bias in units of log 2; a finite one stays finite.
__device__ __forceinline__ float log2_units(float b) {
    const float q = b * kLog2e;
    return __builtin_isfinite(b) ? fminf(fmaxf(q, kLowest), -kLowest) : q;
}

// loss of a row from its maximum, log of the sum and its label's logit, all in units of log 2, and the label's bias.  (m - z) first:
// the loss of a row whose label has nearly all the probability is far below an ulp of lse.  Units of log 2 end at a logit
// of -2.36e38: a bias below that is the label's logit.
__device__ __forceinline__ float row_loss(float m, float ls, float z, float bias) {
    return bias < kLowest * kLn2 ? (m + ls) * kLn2 - bias : ((m - z) + ls) * kLn2;
}

// lse in units of log 2 for the backward, which takes exp2(z - lse) of the forward's z, bit for bit.  Between the two lse has been
// rounded a few times, 2^-22 of it: from 2^21 on that is worth a good part of a unit and more, and lse is raised by 2^-20, so
// that no probability is above 1 (one that overflows the fp16 planes would make the gradient of W infinite for every
// row).
__device__ __forceinline__ float lse_units(float lse) {
    const float l = lse * kLog2e;
    return fabsf(l) >= 0x1p21f ? __builtin_fmaf(fabsf(l), 0x1p-20f, l) : l;
}

// What takes the powers of two out of a row's products and brings them into units of log 2: at most the largest float, so that a
// product of zero stays one; 0 where the operands are too small for any logit to differ from its bias.
__device__ __forceinline__ float logit_unit(int ew, int ex) { return fminf(ldexpf(kLog2e, -ew - ex), -kLowest); }

// The largest of the `parts` partials of quantity `which`.
__device__ __forceinline__ unsigned max_of_parts(const unsigned* __restrict__ part, int which, int parts) {
    unsigned m = 0u, o[kMaxParts / 64];
#pragma unroll
    for (int k = 0; k < kMaxParts / 64; ++k) {                   // all loads in flight at once
        const int i = (threadIdx.x & 63) + 64 * k;
        o[k] = i < parts ? part[which * kMaxParts + i] : 0u;
    }
#pragma unroll
    for (int k = 0; k < kMaxParts / 64; ++k) m = m > o[k] ? m : o[k];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const unsigned q = (unsigned)__shfl_xor((int)m, off, 64);
        m = m > q ? m : q;
    }
    return m;
}

// Exponent field of a float: |d| < 2^(field - 126).
__device__ __forceinline__ int field_of(float d) { return (int)(__builtin_bit_cast(unsigned, d) >> 23 & 0xffu); }

// ---------------------------------------------------------------- planes
__device__ __forceinline__ void split8(const float* v, u32x4& hi, u32x4& lo) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f16x2 h2 = __builtin_convertvector((f32x2){v[2 * k], v[2 * k + 1]}, f16x2);
        hi[k] = __builtin_bit_cast(unsigned, h2);
        lo[k] = f16_pack(v[2 * k] - (float)h2[0], v[2 * k + 1] - (float)h2[1]);
    }
}

struct XentPrep {
    const void* x;
    const float *w, *b, *lse, *dloss;
    const int* labels;
    const unsigned* part;
    int parts;
    long n, v, np, vp;            // rows, classes, and both padded to 128
    int e, ep;                    // features, padded to 128
    f16_t *xh, *xl, *wh, *wl;     // planes: rows x ep, classes x ep
    const unsigned* rmax;         // per labelled row: its largest magnitude
    float* bias;
    // {exponent of W's planes, the largest exponent sum of a row's dloss and x, that of dloss (fields)}
    int* exps;
    // per row: lse (units of log 2), the factor of its dz, the unit of its logits, dloss; (inf, 0, 0, 0) without a label.  A row of x is held
    // under its own power of two 2^ex, so no row's digits depend on another's.  The factor of dz, streamed: dloss 2^-ex, counted
    // from its largest, so that the planes of x times dz sum to dW.  Wide features, where dz is stored and serves dx too:
    // dloss 2^14 over its own power of two, which goes into dx; both powers, counted from the largest, go into
    // the planes of x that dW is made of (xsh, xsl), and dloss's into the weights of db (ones).
    f32x4* row;
    f16_t *xsh, *xsl, *ones;
    int* lab;
    long wtiles, xblocks;
};

// Workgroups 0 .. wtiles-1: a 64 classes x 64 features tile of W, transposed through LDS into the class-major planes;
// the next xblocks: the planes of x; the rest: padded bias, labels and per-row scalars, and the exponents.
template <bool XF32>
__global__ __launch_bounds__(256) void xent_prep_kernel(XentPrep p) {
    const int tid = threadIdx.x;
    if ((long)blockIdx.x < p.wtiles) {
        __shared__ float t[64][65];
        const long etiles = p.ep / 64, ct = blockIdx.x / etiles, et = blockIdx.x - ct * etiles;
        const long c0 = ct * 64, e0 = et * 64;
        const int cc = tid & 63, k0 = tid >> 6;
        const float bc = p.b && c0 + cc < p.v ? p.b[c0 + cc] : 0.f;
        float in[16];                                          // in flight while the exponent is found
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int k = k0 + 4 * j;
            in[j] = c0 + cc < p.v && e0 + k < p.e ? p.w[(e0 + k) * p.v + c0 + cc] : 0.f;
        }
        const int ew = exponent_of(max_of_parts(p.part, 0, p.parts));
#pragma unroll
        for (int j = 0; j < 16; ++j) t[k0 + 4 * j][cc] = masked(bc) ? 0.f : ldexpf(in[j], ew);
        __syncthreads();
        const int e8 = tid & 7;
        for (int c = tid >> 3; c < 64; c += 32) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = t[e8 * 8 + k][c];
            u32x4 hi, lo;
            split8(v, hi, lo);
            const long at = (c0 + c) * p.ep + e0 + e8 * 8;
            *(u32x4*)(p.wh + at) = hi;
            *(u32x4*)(p.wl + at) = lo;
        }
    } else if ((long)blockIdx.x < p.wtiles + p.xblocks) {
        const int most = p.xsh ? (int)max_of_parts(p.part, 1, p.parts) - 1 : 0;
        const int q = p.ep / 8;
        for (long i = ((long)blockIdx.x - p.wtiles) * 256 + tid; i < p.np * q; i += p.xblocks * 256) {
            const long row = i / q;
            const int c = (int)(i - row * q) * 8;
            const int lab = row < p.n ? p.labels[row] : -1;
            const bool ok = lab >= 0 && lab < p.v;
            const long at = row * p.e + c;
            const unsigned rm = ok ? p.rmax[row] : 0u;
            const int ex = exponent_of(rm);
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (ok && (p.e & 7) == 0) {                        // rows of whole 16-byte pieces
                if (c < p.e) {
                    if (XF32) {
                        const f32x4 a = *(const f32x4*)((const float*)p.x + at), b = *(const f32x4*)((const float*)p.x + at + 4);
#pragma unroll
                        for (int k = 0; k < 4; ++k) { v[k] = a[k]; v[4 + k] = b[k]; }
                    } else {
                        const u32x4 a = *(const u32x4*)((const bf16_t*)p.x + at);
#pragma unroll
                        for (int k = 0; k < 4; ++k) { v[2 * k] = bf_lo(a[k]); v[2 * k + 1] = bf_hi(a[k]); }
                    }
                }
            } else if (ok) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (c + k < p.e) v[k] = XF32 ? ((const float*)p.x)[at + k] : (float)((const bf16_t*)p.x)[at + k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k], ex);
            u32x4 hi, lo;
            split8(v, hi, lo);
            *(u32x4*)(p.xh + row * p.ep + c) = hi;
            if (XF32) *(u32x4*)(p.xl + row * p.ep + c) = lo;
            if (p.xsh) {
                const int rel = ok ? field_of(p.dloss[row]) + (int)(rm >> 23) - most : 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k], rel < 0 ? rel : 0);
                split8(v, hi, lo);
                *(u32x4*)(p.xsh + row * p.ep + c) = hi;
                if (XF32) *(u32x4*)(p.xsl + row * p.ep + c) = lo;
            }
        }
    } else {
        const int ew = exponent_of(max_of_parts(p.part, 0, p.parts)), most = (int)max_of_parts(p.part, 1, p.parts) - 1,
                  fd = (int)(max_of_parts(p.part, 2, p.parts) >> 23);
        const long first = (long)blockIdx.x - p.wtiles - p.xblocks, nb = gridDim.x - p.wtiles - p.xblocks;
        if (first == 0 && tid == 0) {
            p.exps[0] = ew;
            p.exps[1] = most;
            p.exps[2] = fd;
        }
        for (long i = first * 256 + tid; i < p.vp; i += nb * 256)
            p.bias[i] = log2_units(i < p.v ? (p.b ? p.b[i] : 0.f) : -__builtin_inff());
        for (long i = first * 256 + tid; i < p.np; i += nb * 256) {
            int lab = i < p.n ? p.labels[i] : -1;
            if (lab < 0 || lab >= p.v) lab = -1;
            p.lab[i] = lab;
            f32x4 info = {__builtin_inff(), 0.f, 0.f, 0.f};       // no label: every exponential of the row is 0
            float weight = 0.f;
            if (lab >= 0) {
                const unsigned rm = p.rmax[i];
                const int ex = exponent_of(rm);
                info[2] = logit_unit(ew, ex);
                if (p.dloss) {
                    const float d = p.dloss[i];
                    const int f = field_of(d);
                    info[0] = lse_units(p.lse[i]);
                    info[1] = p.xsh ? ldexpf(d, 140 - f) : rm ? ldexpf(d, 280 - ex - most) : 0.f;      // a row of zeros adds none to dW
                    info[3] = d;
                    weight = ldexpf(1.f, f < fd ? f - fd : 0);
                }
            }
            p.row[i] = info;
            if (p.ones) p.ones[i] = (f16_t)weight;
        }
    }
}

// ---------------------------------------------------------------- products
// D (64 WM x 64 WN per workgroup of WM x WN = 8 waves) = sum over the kept plane products of A B^T.  An operand is stored either
// with the contraction index fastest ([row][k], read as 16-byte fragments) or slowest ([k][row], read with
// ds_read_b64_tr_b16).  32 of k per step; all planes of a step are staged by LDS-DMA, two steps ahead, into a ring of three: a step is
// 0.4 us of matrix instructions, less than what a load takes under load.  Staged rows have their 16-byte chunks
// XOR-swizzled by the row so that both kinds of read spread over all banks.
constexpr int BK = 32;

struct XentGemm {
    const f16_t *a[2], *b[2];
    long lda, ldb;
    int kiters;
    // epilogues
    const float* bias;
    const int* exps;
    const f32x4* row;
    const int* lab;
    float2* part;
    float *zlab, *out, *outb;
    f16_t *dzh, *dzl;
    long np, ldo, class0;              // class0: first class of the piece
    XentOut o;                         // DW
    const f16_t* ones;                 // DW: what the rows' dz weigh in db
};

enum { EPI_FWD = 0, EPI_DZ = 1, EPI_DX = 2, EPI_DW = 3 };

__device__ __forceinline__ int swz_row(int row) { return (row >> 2) & 3; }
__device__ __forceinline__ int swz_k(int k) { return ((k & 3) << 2) | ((k >> 2) & 3); }

template <int NA, int NB, bool AT, bool BT, int EPI, int WM>
__global__ __launch_bounds__(512, 2) void xent_gemm_kernel(XentGemm g) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    constexpr int WN = 8 / WM, TM = 64 * WM, TN = 64 * WN, PA = TM * BK * 2, PB = TN * BK * 2, BUF = NA * PA + NB * PB;
    constexpr int PIECES = (NA * PA + NB * PB) / 8192;              // LDS-DMA instructions of a wave and step
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5, wm = wv / WN, wn = wv % WN;
    const long m0 = (long)blockIdx.x * TM, n0 = (long)blockIdx.y * TN;
    // split contraction: part z of gridDim.z takes steps [it0, it1)
    const int per = (g.kiters + gridDim.z - 1) / gridDim.z;
    const int it0 = blockIdx.z * per, it1 = it0 + per < g.kiters ? it0 + per : g.kiters;

    // sums of B's columns: a product with the rows' weights
    const bool with_bias = EPI == EPI_DW && blockIdx.x == 0, bias_wave = with_bias && wm == 0;

    // one plane (T rows) of step it: pieces of 1 KB, 16 rows of 64 B or 2 (4) rows of 512 (256) B
    auto stage_plane = [&](unsigned dst, const f16_t* src, long ld, long o0, int it, auto tr_, auto T_) {
        constexpr bool tr = decltype(tr_)::value;
        constexpr int T = decltype(T_)::value, PER = T * BK * 2 / 8192;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int piece = wv * PER + i;
            if constexpr (tr) {
                constexpr int RPP = 512 / T, LPR = 64 / RPP;            // rows of a piece, lanes of a row
                const int row = piece * RPP + lane / LPR, ch = (lane % LPR) ^ swz_k(row);
                lds_dma16(src + ((long)it * BK + piece * RPP) * ld + o0, (int)(lane / LPR * ld * 2) + ch * 16, dst + piece * 1024);
            } else {
                const int ch = (lane & 3) ^ ((lane >> 4) & 3);          // swz_row of row 16 piece + lane / 4
                lds_dma16(src + (o0 + piece * 16) * ld + (long)it * BK, (int)((lane >> 2) * ld * 2) + ch * 16, dst + piece * 1024);
            }
        }
    };
    auto stage = [&](int it) {
        const unsigned dst = lds_byte(lds) + (it - it0) % 3 * BUF;
#pragma unroll
        for (int pl = 0; pl < NA; ++pl)
            stage_plane(dst + pl * PA, g.a[pl], g.lda, m0, it, std::integral_constant<bool, AT>{}, std::integral_constant<int, TM>{});
#pragma unroll
        for (int pl = 0; pl < NB; ++pl)
            stage_plane(dst + NA * PA + pl * PB, g.b[pl], g.ldb, n0, it, std::integral_constant<bool, BT>{}, std::integral_constant<int, TN>{});
        // the rows' weights in db, 64 B behind the ring: every wave writes the same, so that each counts its own loads only
        if (with_bias && lane < 16) lds_dma4(g.ones + (long)it * BK, lane * 4, lds_byte(lds) + 3 * BUF + (it - it0) % 3 * 64);
    };
    const int hk = lane >> 5, cb = (lane >> 4) & 1, qq = (lane >> 2) & 3, pp = lane & 3;
    auto frag = [&](const unsigned char* plane, bool tr, int rowb, int blk, int ks) -> u32x4 {
        if (tr) {
            const int k = 16 * ks + 8 * hk + qq, ch = blk * 4 + 2 * cb + (pp >> 1);
            const u32x2 a = tr_read(plane + k * rowb + ((ch ^ swz_k(k)) << 4) + 8 * (pp & 1));
            const u32x2 b = tr_read(plane + (k + 4) * rowb + ((ch ^ swz_k(k + 4)) << 4) + 8 * (pp & 1));
            return (u32x4){a[0], a[1], b[0], b[1]};
        }
        const int row = blk * 32 + r;
        return *(const u32x4*)(plane + row * 64 + (((2 * ks + h) ^ swz_row(row)) << 4));
    };

    f32x16 acc[2][2], accb[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        acc[0][0][i] = acc[0][1][i] = acc[1][0][i] = acc[1][1][i] = 0.f;
        accb[0][i] = accb[1][i] = 0.f;
    }
    if (it0 < it1) stage(it0);
    if (it0 + 1 < it1) stage(it0 + 1);
    for (int it = it0; it < it1; ++it) {
        // step it has landed (the one behind it may be on its way), and no wave reads step it - 1 any more
        if (it + 1 < it1) {
            if (with_bias) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES + 1) : "memory");
            else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES) : "memory");
        }
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (it + 2 < it1) stage(it + 2);
        const unsigned char* base = lds + (it - it0) % 3 * BUF;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            u32x4 fa[NA][2], fb[NB][2];
#pragma unroll
            for (int pl = 0; pl < NA; ++pl)
#pragma unroll
                for (int i = 0; i < 2; ++i) fa[pl][i] = frag(base + pl * PA, AT, TM * 2, wm * 2 + i, ks);
#pragma unroll
            for (int pl = 0; pl < NB; ++pl)
#pragma unroll
                for (int i = 0; i < 2; ++i) fb[pl][i] = frag(base + NA * PA + pl * PB, BT, TN * 2, wn * 2 + i, ks);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (NA > 1) acc[i][j] = mfma_f16(fa[NA - 1][i], fb[0][j], acc[i][j]);
                    if (NB > 1) acc[i][j] = mfma_f16(fa[0][i], fb[NB - 1][j], acc[i][j]);
                    acc[i][j] = mfma_f16(fa[0][i], fb[0][j], acc[i][j]);
                }
            if (bias_wave) {
                const u32x4 ones = *(const u32x4*)(lds + 3 * BUF + (it - it0) % 3 * 64 + 32 * ks + 16 * h);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (NB > 1) accb[j] = mfma_f16(ones, fb[NB - 1][j], accb[j]);
                    accb[j] = mfma_f16(ones, fb[0][j], accb[j]);
                }
            }
        }
    }

    const long mw = m0 + wm * 64, nw = n0 + wn * 64;
    if constexpr (EPI == EPI_FWD || EPI == EPI_DZ) {
        // A: classes, B: rows of x
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const long row = nw + j * 32 + r;
            const int lab = g.lab[row];
            const f32x4 info = g.row[row];
            const float unit = info[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 bv = *(const f32x4*)(g.bias + mw + i * 32 + 8 * q + 4 * h);
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[i][j][4 * q + k] = __builtin_fmaf(acc[i][j][4 * q + k], unit, bv[k]);
                }
            const long rel = lab - g.class0 - mw;           // the label's place among the wave's 64 classes
            if constexpr (EPI == EPI_FWD) {
                float m = kLowest, s = 0.f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int k = 0; k < 16; ++k) m = fmaxf(m, acc[i][j][k]);
                m = fmaxf(m, __shfl_xor(m, 32, 64));
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int k = 0; k < 16; ++k) s += __builtin_amdgcn_exp2f(acc[i][j][k] - m);
                s += __shfl_xor(s, 32, 64);
                if (h == 0) g.part[(mw / 64) * g.np + row] = make_float2(m, s);
                if (lab >= 0 && rel >= 0 && rel < 64) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (i * 32 + (k & 3) + 8 * (k >> 2) + 4 * h == (int)rel) g.zlab[row] = acc[i][j][k];
                }
            } else {
                const float lse = info[0], dl = info[1];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float p = __builtin_amdgcn_exp2f(acc[i][j][k] - lse);
                        if (i * 32 + (k & 3) + 8 * (k >> 2) + 4 * h == rel) p -= 1.f;           // no label: rel < 0
                        acc[i][j][k] = p * dl;
                    }
                    acc_rows_interleaved(acc[i][j]);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = acc[i][j][8 * half + k];
                        u32x4 hi, lo;
                        split8(v, hi, lo);
                        const long at = row * g.ldo + mw + i * 32 + 16 * half + 8 * h;
                        *(u32x4*)(g.dzh + at) = hi;
                        *(u32x4*)(g.dzl + at) = lo;
                    }
                }
            }
        }
    } else if constexpr (EPI == EPI_DX) {
        // A: rows, B: features; slab z, which the pieces of the classes add to one after the other
        float* out = g.out + (long)blockIdx.z * g.np * g.ldo;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    float* o = out + (mw + i * 32 + acc_row(k, lane)) * g.ldo + nw + j * 32 + r;
                    *o = g.class0 == 0 ? acc[i][j][k] : *o + acc[i][j][k];
                }
    } else {
        // A: features, B: classes; the gradients, or slab z of the piece
        if (g.o.direct) {
            const int ed = g.exps[1] - 280, eb = g.exps[2] - 140;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const long c = nw + j * 32 + r;
                if (c >= g.o.cnt) continue;
                if (g.o.dw) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const long f = mw + i * 32 + acc_row(k, lane);
                            if (f < g.o.e) {
                                float* d = g.o.dw + f * g.o.v + c;
                                const float q = ldexpf(acc[i][j][k], ed);
                                *d = g.o.accumulate ? *d + q : q;
                            }
                        }
                }
                if (bias_wave && h == 0 && g.o.db) {
                    const float q = ldexpf(accb[j][0], eb);
                    g.o.db[c] = g.o.accumulate ? g.o.db[c] + q : q;
                }
            }
            return;
        }
        float* out = g.out + (long)blockIdx.z * g.np;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k) out[(mw + i * 32 + acc_row(k, lane)) * g.ldo + nw + j * 32 + r] = acc[i][j][k];
        if (bias_wave && h == 0) {
#pragma unroll
            for (int j = 0; j < 2; ++j) g.outb[(long)blockIdx.z * g.ldo + nw + j * 32 + r] = accb[j][0];
        }
    }
}

// ---------------------------------------------------------------- narrow features
// Up to EP features (EP = 64 or 128) the two products around the exponential run in one kernel and no dz is stored.  One operand is
// resident: a wave keeps 32 RB of its items (rows of x, or classes) as B fragments in registers.  The other is streamed: tiles of
// 32 of its items in LDS, a ring of four filled by LDS-DMA and shared by the four waves.  Per streamed tile:
//     S (32 streamed x 32 RB resident) = sum over plane products                         first product; logits: S unit + bias
//     forward: the lane's running maximum and sum over the streamed classes
//     backward: P = exp(S - lse) (times dloss where rows are streamed) - label, as fp16 planes: the accumulator registers
//               8 t .. 8 t + 7 of a lane are the streamed items 16 t + 4 h + {0..3} and 16 t + 8 + 4 h + {0..3}, which is the
//               B fragment of a product over 16 streamed items taken in that order
//     D (EP x 32 RB) += streamed^T P, the A fragments read transposed (ds_read_b64_tr_b16) from the same tile in that order
// The three run as a pipeline, one step a tile: S of tile i + 1, the exponentials of tile i and D of tile i - 1 do not depend on
// each other.  A step is a fixed sequence of units, each the matrix instructions of one A fragment (read from LDS two units
// ahead) with a piece of the exponentials, pinned by scheduling barriers: left to itself the compiler moves all LDS reads of a step to
// its front and spills the resident fragments.  The labels of a tile are few and are put in behind its step: P is formed
// again with the comparisons (a branch around two whole copies of the step costs 100 registers of copies where they meet).
// MODE FWD and DX: rows resident, classes streamed; DW: classes resident, rows streamed.  gridDim.y parts of the streamed
// operand leave partial results that are joined in order.
// DX of a bf16 x (NR = 1), whose result is rounded to 8 bits, takes one plane of W and one of P in the second product, 2^-11 of a
// term each.  The logits take both planes of W: an exponential turns a logit's absolute error into a relative one, and
// one plane, 2^-11 of the logit's terms, would be off by more than the result's rounding for logits of a few units.
enum { MODE_FWD = 0, MODE_DX = 1, MODE_DW = 2 };
constexpr int ST = 32;                              // streamed items of a tile

struct XentStream {
    const f16_t *r[2], *s[2];
    const int* exps;
    const float* bias;                              // classes
    const f32x4* row;                               // rows: lse, factor of dz, unit, dloss
    const int* lab;                                 // rows
    int tiles;                                      // streamed tiles
    float2* part;                                   // FWD: (maximum, sum) per part and row
    float* zlab;                                    // FWD
    float* out;                                     // DX: part x rows x EP; DW: part x EP x classes
    float* outb;                                    // DW: part x classes
    long ld;                                        // rows (FWD, DX) or classes (DW), padded
    XentOut o;                                      // DW
};

template <int EP>
__device__ __forceinline__ int swz_item(int row) {
    return EP == 64 ? ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) : (((row & 3) << 2) | ((row >> 2) & 3));
}

template <int EP, int NR, int NS, int RB, int MODE, int OCC>
__global__ __launch_bounds__(256, OCC) void xent_stream_kernel(XentStream g) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    constexpr int KS = EP / 16, EB = EP / 32, ROWB = EP * 2, SPLANE = ST * ROWB;
    constexpr int BUF = NS * SPLANE + 1024;
    // Plane of unit si of S.  The products of a logit are added in one order in every mode (x lo W hi, x hi W hi, x hi W lo): the backward
    // meets the bits of the forward's logits, so that exp(z - lse) is above 1 by the rounding of lse only, whatever the terms cancel.
    constexpr auto s_plane = [](int si) constexpr { return MODE == MODE_DW ? NS - 1 - si % NS : si % NS; };
    constexpr int NP = MODE == MODE_DW ? 2 : NR;    // planes of P: DX of a bf16 x needs one (its result is rounded to 8 bits)
    constexpr int NA = MODE == MODE_DW ? NS : NR;   // planes of the streamed operand in the second product
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int item0 = (int)(blockIdx.x * 4 + wv) * (32 * RB);
    const int per = (g.tiles + gridDim.y - 1) / gridDim.y;
    const int t0 = blockIdx.y * per, t1 = t0 + per < g.tiles ? t0 + per : g.tiles;

    // LDS-DMA of tile t: a wave fills 1 KB pieces (4 rows of 256 B or 8 of 128 B), lane l the 16-byte place l of the piece with
    // the chunk that belongs there: the swizzle of the lane's row in the first piece, and a bit that is uniform in later ones.
    // In assembly: in front of a transposed LDS read the compiler waits for every LDS-DMA it knows of, the one just issued
    // for a later tile included.
    // beside the planes: FWD and DX the biases (128 B, twice), DW what the rows have (512 B) and their labels
    const float* ip = MODE != MODE_DW ? g.bias : wv < 2 ? (const float*)g.row + 64 * wv : (const float*)g.lab;
    const int lrow = EP == 128 ? lane >> 4 : lane >> 3;
    const int lo0 = lrow * ROWB + (((lane & (EP / 8 - 1)) ^ swz_item<EP>(lrow)) << 4);
    auto stage = [&](int t) {
        const unsigned dst = lds_byte(lds) + (t & 3) * BUF;
        constexpr int PIECES = SPLANE / 1024;
#pragma unroll
        for (int pl = 0; pl < NS; ++pl)
#pragma unroll
            for (int i = 0; i < PIECES / 4; ++i) {
                const int piece = wv * (PIECES / 4) + i, flip = EP == 128 ? (piece & 3) << 4 : (piece & 1) << 5;
                lds_dma16(g.s[pl] + ((long)t * SPLANE + piece * 1024) / 2, lo0 ^ flip, dst + pl * SPLANE + piece * 1024);
            }
        if (wv < (MODE == MODE_DW ? 3 : 1)) {        // 64 floats, or 32 twice
            const bool half = MODE == MODE_DW && wv < 2;
            lds_dma4(ip + (long)t * (half ? 4 * ST : ST), half ? lane * 4 : r * 4, dst + NS * SPLANE + wv * 256);
        }
    };

    if (t0 < t1) stage(t0);
    if (t0 + 1 < t1) stage(t0 + 1);

    // resident fragments: lane r's item, features 16 ks + 8 h .. + 7
    u32x4 fb[NR][RB][KS];
#pragma unroll
    for (int pl = 0; pl < NR; ++pl)
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                fb[pl][b][ks] = *(const u32x4*)(g.r[pl] + ((long)item0 + 32 * b + r) * EP + 16 * ks + 8 * h);
    float unit[RB];                                 // FWD, DX
    float rinfo[RB];                                // DX: -(lse - 14); DW: bias
    int rlab[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const long it = item0 + 32 * b + r;
        rinfo[b] = MODE == MODE_DW ? g.bias[it] : MODE == MODE_DX ? 14.f - g.row[it][0] : 0.f;
        unit[b] = MODE == MODE_DW ? 0.f : g.row[it][2];
        rlab[b] = MODE == MODE_DW ? 0 : g.lab[it];
    }
    // LDS offsets of the lane: the first fragment of its row, and the first transposed reads.  A row starts at a multiple of
    // its size and the swizzle is an XOR, so further fragments (feature blocks) are an XOR of 32 ks (64 eb) away.
    const int cb = (lane >> 4) & 1, qq = (lane >> 2) & 3, pp = lane & 3;
    int ao = r * ROWB + ((h ^ swz_item<EP>(r)) << 4);
    int to[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = 8 * j + 4 * h + qq;
        to[j] = row * ROWB + (((2 * cb + (pp >> 1)) ^ swz_item<EP>(row)) << 4) + 8 * (pp & 1);
    }

    float m[RB], ssum[RB];
    f32x16 dacc[MODE == MODE_FWD ? 1 : EB][RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        m[b] = kLowest;
        ssum[b] = 0.f;
#pragma unroll
        for (int eb = 0; eb < (MODE == MODE_FWD ? 1 : EB); ++eb)
#pragma unroll
            for (int i = 0; i < 16; ++i) dacc[eb][b][i] = 0.f;
    }

    // whether tile t holds a label of this wave's resident items (rows resident: a lane's own label; classes: the rows' labels)
    auto labels_in = [&](int t) -> bool {
        bool in = false;
        if constexpr (MODE == MODE_DW) {
            const int lb = *(const int*)(lds + (t & 3) * BUF + NS * SPLANE + 512 + r * 4);
            in = lb >= item0 && lb < item0 + 32 * RB;
        } else {
#pragma unroll
            for (int b = 0; b < RB; ++b) in = in || (unsigned)(rlab[b] - t * ST) < (unsigned)ST;
        }
        return __ballot(in) != 0;
    };
    // one barrier a step: tile i + 1 has landed for every wave, and none reads tile i - 2 any more, whose place tile i + 2 takes
    auto arrive = [&](int i) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (i + 2 < t1) stage(i + 2);
    };
    // units of a step: NSU fragments of S (feature step, plane) and NGU of D (16 items, feature block, plane), evenly mixed with D first
    constexpr int NSU = KS * NS, NGU = MODE == MODE_FWD ? 0 : 2 * EB * NA, NU = NSU + NGU;
    constexpr int PB = MODE == MODE_FWD ? 9 : 8, NPIECE = PB * RB;         // pieces: pairs of values (FWD: the maximum first)
    // PART 1: S only (in front of the first tile); 2: S and the exponentials; 3: all; 4: D only (behind the last tile)
    auto step = [&](int i, f32x16 (&cur)[RB], f32x16 (&nxt)[RB], u32x4 (&fcur)[NP][RB][2], u32x4 (&fprev)[NP][RB][2], auto part) {
        constexpr int PART = decltype(part)::value;
        constexpr bool DO_S = PART != 4, DO_E = PART == 2 || PART == 3, DO_G = PART >= 3;
        const unsigned char* ts = lds + ((i + 1) & 3) * BUF;
        const unsigned char* te = lds + (i & 3) * BUF + NS * SPLANE;
        const unsigned char* tg = lds + ((i - 1) & 3) * BUF;
        asm volatile("" : "+v"(ao), "+v"(to[0]), "+v"(to[1]));      // keeps the 16 addresses derived from them out of registers
        const int s0 = i * ST;
        u32x4 fr[3];
        f32x4 ri2[2];                                // DW: what the two rows of the next pair have
        f32x2 bi2;                                   // DX: biases of the next pair
        f32x4 bv[4];                                 // FWD: biases of the tile
        float tsum[RB];                              // DW: the tile's sum of P, added to the running one once a tile
#pragma unroll
        for (int b = 0; b < RB; ++b) tsum[b] = 0.f;
        auto load = [&](auto U_) {
            constexpr int u = decltype(U_)::value;
            if constexpr (u < NU) {
                constexpr int gc = (u * NGU + NU - 1) / NU;
                if constexpr (((u + 1) * NGU + NU - 1) / NU > gc) {
                    constexpr int x = gc / (EB * NA), eb = gc % (EB * NA) / NA, pl = NA - 1 - gc % NA;
                    if constexpr (DO_G) {
                        const unsigned char* tp = tg + pl * SPLANE + x * 16 * ROWB;
                        const u32x2 a0 = tr_read(tp + (to[0] ^ (eb << 6))), a1 = tr_read(tp + (to[1] ^ (eb << 6)));
                        fr[u % 3] = (u32x4){a0[0], a0[1], a1[0], a1[1]};
                    }
                } else if constexpr (DO_S) {
                    constexpr int si = u - gc, ks = si / NS, pl = s_plane(si);
                    fr[u % 3] = *(const u32x4*)(ts + pl * SPLANE + (ao ^ (ks << 5)));
                }
            }
        };
        auto products = [&](auto U_) {
            constexpr int u = decltype(U_)::value, gc = (u * NGU + NU - 1) / NU;
            if constexpr (((u + 1) * NGU + NU - 1) / NU > gc) {
                constexpr int x = gc / (EB * NA), eb = gc % (EB * NA) / NA, pl = NA - 1 - gc % NA;
                if constexpr (DO_G) {
#pragma unroll
                    for (int b = 0; b < RB; ++b) {
                        if constexpr (NP > 1 && pl == 0) dacc[eb][b] = mfma_f16(fr[u % 3], fprev[NP - 1][b][x], dacc[eb][b]);
                        dacc[eb][b] = mfma_f16(fr[u % 3], fprev[0][b][x], dacc[eb][b]);
                    }
                }
            } else if constexpr (DO_S) {
                constexpr int si = u - gc, ks = si / NS, pl = s_plane(si);
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    if constexpr (MODE != MODE_DW && NR > 1 && pl == 0) nxt[b] = mfma_f16(fr[u % 3], fb[NR - 1][b][ks], nxt[b]);
                    nxt[b] = mfma_f16(fr[u % 3], fb[0][b][ks], nxt[b]);
                    if constexpr (MODE == MODE_DW && NR > 1 && pl == 0) nxt[b] = mfma_f16(fr[u % 3], fb[NR - 1][b][ks], nxt[b]);
                }
            }
        };
        // a pair of P as fp16 planes (piece p: pair p / RB of resident item block p % RB)
        auto put = [&](auto P_, float v0, float v1) {
            constexpr int p = decltype(P_)::value, b = p % RB, j = p / RB;
            const f16x2 h2 = __builtin_convertvector((f32x2){v0, v1}, f16x2);
            fcur[0][b][j >> 2][j & 3] = __builtin_bit_cast(unsigned, h2);
            if constexpr (NP > 1) fcur[NP - 1][b][j >> 2][j & 3] = f16_pack(v0 - (float)h2[0], v1 - (float)h2[1]);
        };
        // what streamed row k of pair j has
        auto row2 = [&](int j, int k) { return *(const f32x4*)(te + (8 * (j >> 1) + 4 * h + 2 * (j & 1) + k) * 16); };
        // biases of the two streamed classes of pair j
        auto bias2 = [&](int j) { return *(const f32x2*)(te + (8 * (j >> 1) + 4 * h + 2 * (j & 1)) * 4); };
        auto piece = [&](auto P_) {
            constexpr int p = decltype(P_)::value, b = MODE == MODE_FWD ? p / PB : p % RB, j = MODE == MODE_FWD ? p % PB - 1 : p / RB;
            if constexpr (MODE == MODE_FWD && j < 0) {
                float mm = m[b];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    cur[b][k] = __builtin_fmaf(cur[b][k], unit[b], bv[k >> 2][k & 3]);
                    mm = fmaxf(mm, cur[b][k]);
                }
                ssum[b] *= __builtin_amdgcn_exp2f(m[b] - mm);
                m[b] = mm;
            } else if constexpr (MODE == MODE_FWD) {
#pragma unroll
                for (int k = 2 * j; k < 2 * j + 2; ++k) ssum[b] += __builtin_amdgcn_exp2f(cur[b][k] - m[b]);
            } else if constexpr (MODE == MODE_DX) {
                const f32x2 q = bi2;
                const float v0 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[b][2 * j], unit[b], q[0]) + rinfo[b]);
                const float v1 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[b][2 * j + 1], unit[b], q[1]) + rinfo[b]);
                if constexpr (b == RB - 1 && j < 7) bi2 = bias2(j + 1);
                put(P_, v0, v1);
            } else {
                const f32x4 q0 = ri2[0], q1 = ri2[1];
                const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[b][2 * j], q0[2], rinfo[b]) - q0[0]), v0 = e0 * q0[1];
                const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[b][2 * j + 1], q1[2], rinfo[b]) - q1[0]), v1 = e1 * q1[1];
                tsum[b] = __builtin_fmaf(e1, q1[3], __builtin_fmaf(e0, q0[3], tsum[b]));
                if constexpr (b == RB - 1 && j < 7) {
                    ri2[0] = row2(j + 1, 0);
                    ri2[1] = row2(j + 1, 1);
                }
                put(P_, v0, v1);
            }
        };
        // the labels of tile i: FWD keeps their logits, DX and DW form P again
        auto label_piece = [&](auto P_) {
            constexpr int p = decltype(P_)::value, b = MODE == MODE_FWD ? p / 8 : p % RB, j = MODE == MODE_FWD ? p % 8 : p / RB, k = 2 * j, c0 = (k & 3) + 8 * (k >> 2);
            if constexpr (MODE == MODE_FWD) {
                const int rel = rlab[b] - s0 - 4 * h;
                if (rel == c0) g.zlab[item0 + 32 * b + r] = cur[b][k];
                if (rel == c0 + 1) g.zlab[item0 + 32 * b + r] = cur[b][k + 1];
            } else if constexpr (MODE == MODE_DX) {
                const int rel = rlab[b] - s0 - 4 * h;
                const f32x2 q = bias2(j);
                const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[b][k], unit[b], q[0]) + rinfo[b]);
                const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[b][k + 1], unit[b], q[1]) + rinfo[b]);
                put(P_, rel == c0 ? e0 - kDz : e0, rel == c0 + 1 ? e1 - kDz : e1);
            } else {
                const f32x4 q0 = row2(j, 0), q1 = row2(j, 1);
                const u32x2 lb = *(const u32x2*)(te + 512 + (c0 + 4 * h) * 4);
                const bool is0 = (int)lb[0] - item0 - 32 * b == r, is1 = (int)lb[1] - item0 - 32 * b == r;
                const float d0 = is0 ? q0[1] : 0.f, d1 = is1 ? q1[1] : 0.f;
                tsum[b] -= (is0 ? q0[3] : 0.f) + (is1 ? q1[3] : 0.f);
                // (p - 1) times the factor, as one fma each: p times it would have lost the digits of a p next to 1
                const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[b][k], q0[2], rinfo[b]) - q0[0]);
                const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[b][k + 1], q1[2], rinfo[b]) - q1[0]);
                put(P_, __builtin_fmaf(e0, q0[1], -d0), __builtin_fmaf(e1, q1[1], -d1));
            }
        };
        if constexpr (DO_S) {
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int k = 0; k < 16; ++k) nxt[b][k] = 0.f;
        }
        if constexpr (DO_E && MODE == MODE_FWD) {
#pragma unroll
            for (int q = 0; q < 4; ++q) bv[q] = *(const f32x4*)(te + (8 * q + 4 * h) * 4);
        }
        if constexpr (DO_E && MODE == MODE_DX) {
            bi2 = bias2(0);
        }
        if constexpr (DO_E && MODE == MODE_DW) {
            ri2[0] = row2(0, 0);
            ri2[1] = row2(0, 1);
        }
        load(std::integral_constant<int, 0>{});
        load(std::integral_constant<int, 1>{});
        static_for<0, NU>([&](auto U_) {
            constexpr int u = decltype(U_)::value;
            load(std::integral_constant<int, u + 2>{});
            products(U_);
            if constexpr (DO_E) static_for<u * NPIECE / NU, (u + 1) * NPIECE / NU>(piece);
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (DO_E) {
            if (labels_in(i)) static_for<0, 8 * RB>(label_piece);
            if constexpr (MODE == MODE_DW) {
#pragma unroll
                for (int b = 0; b < RB; ++b) ssum[b] += tsum[b];
            }
        }
    };
    using P1 = std::integral_constant<int, 1>;
    using P2 = std::integral_constant<int, 2>;
    using P3 = std::integral_constant<int, 3>;
    using P4 = std::integral_constant<int, 4>;

    if (t0 < t1) {
        f32x16 a0[RB], a1[RB];
        u32x4 p0[NP][RB][2], p1[NP][RB][2];
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        step(t0 - 1, a1, a0, p1, p0, P1{});
        // the S of a step past the last tile works on a stale buffer and is not used
        auto full = [&](int i, f32x16 (&cur)[RB], f32x16 (&nxt)[RB], u32x4 (&fcur)[NP][RB][2], u32x4 (&fprev)[NP][RB][2], auto part) {
            arrive(i);
            step(i, cur, nxt, fcur, fprev, part);
        };
        full(t0, a0, a1, p0, p1, P2{});
        int i = t0 + 1;
        for (; i + 1 < t1; i += 2) {
            full(i, a1, a0, p1, p0, P3{});
            full(i + 1, a0, a1, p0, p1, P3{});
        }
        if (i < t1) {
            full(i, a1, a0, p1, p0, P3{});
            step(i + 1, a0, a1, p0, p1, P4{});
        } else {
            step(i, a1, a0, p1, p0, P4{});
        }
    }

#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const long it = item0 + 32 * b + r;
        if constexpr (MODE == MODE_FWD) {
            const float mo = __shfl_xor(m[b], 32, 64), so = __shfl_xor(ssum[b], 32, 64);
            const float mm = fmaxf(m[b], mo);
            const float s = ssum[b] * __builtin_amdgcn_exp2f(m[b] - mm) + so * __builtin_amdgcn_exp2f(mo - mm);
            if (h == 0) g.part[(long)blockIdx.y * g.ld + it] = make_float2(mm, s);
        } else if constexpr (MODE == MODE_DX) {
            float* o = g.out + ((long)blockIdx.y * g.ld + it) * EP;
#pragma unroll
            for (int eb = 0; eb < EB; ++eb)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(f32x4*)(o + 32 * eb + 8 * q + 4 * h) =
                        (f32x4){dacc[eb][b][4 * q], dacc[eb][b][4 * q + 1], dacc[eb][b][4 * q + 2], dacc[eb][b][4 * q + 3]};
        } else {
            const float so = __shfl_xor(ssum[b], 32, 64);
            if (g.o.direct) {
                if (it >= g.o.cnt) continue;
                const int ed = g.exps[1] - 280;
                if (g.o.dw) {
#pragma unroll
                    for (int eb = 0; eb < EB; ++eb)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int f = 32 * eb + acc_row(i, lane);
                            if (f < g.o.e) {
                                float* d = g.o.dw + f * g.o.v + it;
                                const float q = ldexpf(dacc[eb][b][i], ed);
                                *d = g.o.accumulate ? *d + q : q;
                            }
                        }
                }
                if (h == 0 && g.o.db) {
                    const float q = ssum[b] + so;
                    g.o.db[it] = g.o.accumulate ? g.o.db[it] + q : q;
                }
                continue;
            }
            float* o = g.out + (long)blockIdx.y * EP * g.ld + it;
#pragma unroll
            for (int eb = 0; eb < EB; ++eb)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[(32 * eb + acc_row(i, lane)) * g.ld] = dacc[eb][b][i];
            if (h == 0) g.outb[(long)blockIdx.y * g.ld + it] = ssum[b] + so;
        }
    }
}

// p[0] + p[stride] + ... of n parts, in order, eight loads in flight
__device__ __forceinline__ float sum_parts(const float* __restrict__ p, int n, long stride) {
    float s = 0.f;
    for (int z = 0; z < n; z += 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = z + k < n ? p[(z + k) * stride] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += v[k];
    }
    return s;
}

// dx from its parts in G groups of consecutive parts, then the groups in order: one group where the outputs fill the chip, sixteen
// where they are few and the parts many
struct XentDxJoin {
    const float* parts;
    const int* exps;               // NULL: the parts are those of dx itself
    const f32x4* row;
    bool wide;
    void* dx;
    int dx_f32, np;
    long part, n;
    int e, ep;
};

template <int G>
__device__ __forceinline__ void xent_dx_join(const XentDxJoin& j, long block, long blocks) {
    constexpr int W = G == 1 ? 256 : 64;
    __shared__ float red[G][G == 1 ? 1 : 64];
    const auto [parts, exps, rowinfo, wide, dx, dx_f32, np, part, n, e, ep] = j;
    // streamed: the parts are of 2^14 dz / dloss; wide: of 2^14 dz over the power of two of dloss
    const int ew = exps ? exps[0] : 0;
    const int lane = threadIdx.x % W, q = threadIdx.x / W;
    const int per = (np + G - 1) / G, p0 = q * per, cnt = np - p0 < per ? np - p0 : per;
    for (long i = block * W + lane; i - lane < n * ep; i += blocks * W) {
        float s = i < n * ep && cnt > 0 ? sum_parts(parts + p0 * part + i, cnt, part) : 0.f;
        if constexpr (G > 1) {
            __syncthreads();
            red[q][lane] = s;
            __syncthreads();
            if (q == 0)
                for (int k = 1; k < G; ++k) s += red[k][lane];
        }
        const long row = i / ep;
        const int c = (int)(i - row * ep);
        if (q == 0 && row < n && c < e) {
            if (exps) {
                const float d = rowinfo[row][3];
                const int f = field_of(d);
                s = ldexpf(wide ? s : s * ldexpf(d, 126 - f), f - 140 - ew);
            }
            if (dx_f32) ((float*)dx)[row * e + c] = s;
            else ((bf16_t*)dx)[row * e + c] = (bf16_t)s;
        }
    }
}

template <int G>
__global__ __launch_bounds__(G == 1 ? 256 : 1024) void xent_dx_join_kernel(XentDxJoin j) {
    xent_dx_join<G>(j, blockIdx.x, gridDim.x);
}

// loss and lse of 32 rows per workgroup from the partial (maximum, sum) of the parts or of every 64 classes
__global__ __launch_bounds__(256) void xent_join_kernel(const float2* __restrict__ part, const float* __restrict__ zlab,
                                                        const float* __restrict__ b, const int* __restrict__ lab, float* __restrict__ loss,
                                                        float* __restrict__ lse, int* __restrict__ hits, long n, long np,
                                                        long slices) {
    __shared__ float2 red[8][32];
    const int rr = threadIdx.x & 31, gr = threadIdx.x >> 5;
    const long row = (long)blockIdx.x * 32 + rr;
    float m = kLowest, s = 0.f;
    for (long i = gr; i < slices; i += 32) {                     // four loads in flight
        float2 p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = i + 8 * k < slices ? part[(i + 8 * k) * np + row] : make_float2(kLowest, 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float mm = fmaxf(m, p[k].x);
            s = s * __builtin_amdgcn_exp2f(m - mm) + p[k].y * __builtin_amdgcn_exp2f(p[k].x - mm);
            m = mm;
        }
    }
    red[gr][rr] = make_float2(m, s);
    __syncthreads();
    if (gr == 0 && row < n) {
        for (int q = 1; q < 8; ++q) {
            const float2 p = red[q][rr];
            const float mm = fmaxf(m, p.x);
            s = s * __builtin_amdgcn_exp2f(m - mm) + p.y * __builtin_amdgcn_exp2f(p.x - mm);
            m = mm;
        }
        const bool ok = lab[row] >= 0;
        const float ls = __builtin_amdgcn_logf(s);
        loss[row] = ok ? row_loss(m, ls, zlab[row], b ? b[lab[row]] : 0.f) : 0.f;
        lse[row] = ok ? (m + ls) * kLn2 : 0.f;
        if (hits) hits[row] = ok && zlab[row] >= m ? 1 : 0;
    }
}

// dW and db of a piece of the classes from the slabs of the split contraction, in order: 256 classes of a feature (or of db) a block
struct XentDwReduce {
    const float *slabs, *slabs_b;
    const int* exps;
    bool wide;                         // slabs_b under the largest dloss's power of two
    float *dw, *db;
    int nz;
    long slab, ldo;
    int e;
    long v, c0, cnt;                   // classes of W, first class, classes of the piece
    int accumulate;
    long blocks() const { return (cnt + 255) / 256 * (e + 1); }
};

__device__ __forceinline__ void xent_dw_reduce(const XentDwReduce& g, long block) {
    const long cols = (g.cnt + 255) / 256, k = block / cols, c = (block - k * cols) * 256 + threadIdx.x;
    if (c >= g.cnt || g.c0 + c >= g.v) return;
    if (k < g.e) {
        if (!g.dw) return;
        const float s = ldexpf(sum_parts(g.slabs + k * g.ldo + c, g.nz, g.slab), g.exps[1] - 280);
        float* d = g.dw + k * g.v + g.c0 + c;
        *d = g.accumulate ? *d + s : s;
    } else if (g.db) {
        const float all = sum_parts(g.slabs_b + c, g.nz, g.ldo), s = g.wide ? ldexpf(all, g.exps[2] - 140) : all;
        float* d = g.db + g.c0 + c;
        *d = g.accumulate ? *d + s : s;
    }
}

__global__ __launch_bounds__(256) void xent_dw_reduce_kernel(XentDwReduce g) { xent_dw_reduce(g, blockIdx.x); }

// both in one launch: the first `blocks` workgroups join dx
__global__ __launch_bounds__(256) void xent_joins_kernel(XentDxJoin j, long blocks, XentDwReduce g) {
    if ((long)blockIdx.x < blocks) xent_dx_join<1>(j, blockIdx.x, blocks);
    else xent_dw_reduce(g, blockIdx.x - blocks);
}

// ---------------------------------------------------------------- few rows
// Few rows: the kernel W is what the call reads and dW what it writes: float32 on the vector ALU, no planes, two launches a
// direction.  A workgroup takes 64 classes (a lane each, so a wave reads 256 consecutive bytes of a row of W), its four
// waves a quarter of the features each.  RT: rows rounded up (1, 4, 16), accumulators of a lane: 4 x 128 x 65536 takes 15 + 42 us
// with 4 and 18 + 65 with 16, 1 x 128 x 4097 15 + 17 with 1 and 16 + 20 with 16.
constexpr int FEW = 16, RC = 256;                   // RC: features staged at a time

struct XentRows {
    const void* x;
    const float *w, *b, *lse, *dloss;
    const int* labels;
    float2* part;                                   // forward: (maximum, sum) per 64 classes and row
    float* zlab;
    float *dxp, *dw, *db;                           // backward: dx per 64 classes, row and feature; gradients
    long v;
    int n, e, accumulate;
};

// xs[RT][RC]: features e0 .. of the rows that have a label, zeros elsewhere
template <int RT, bool XF32>
__device__ __forceinline__ void xent_rows_stage(const XentRows& g, float* xs, int e0, int cnt) {
    for (int k = threadIdx.x; k < RT * RC; k += 256) {
        const int i = k / RC, c = k - i * RC;
        float v = 0.f;
        if (i < g.n && c < cnt) {
            const int lab = g.labels[i];
            const long at = (long)i * g.e + e0 + c;
            if (lab >= 0 && lab < g.v) v = XF32 ? ((const float*)g.x)[at] : (float)((const bf16_t*)g.x)[at];
        }
        xs[k] = v;
    }
}

// zs[RT][64]: the logits of the workgroup's classes in units of log 2
template <int RT, bool XF32>
__device__ __forceinline__ void xent_rows_logits(const XentRows& g, float* xs, float* red, float* zs) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const long c = (long)blockIdx.x * 64 + lane;
    const bool ok = c < g.v;
    float z[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) z[i] = 0.f;
    for (int e0 = 0; e0 < g.e; e0 += RC) {
        const int cnt = g.e - e0 < RC ? g.e - e0 : RC;
        __syncthreads();
        xent_rows_stage<RT, XF32>(g, xs, e0, cnt);
        __syncthreads();
        const int per = (cnt + 63) / 64 * 16, k1 = (wv + 1) * per < cnt ? (wv + 1) * per : cnt;
        for (int k = wv * per; k < k1; k += 16) {                  // 16 loads in flight; k + 15 < RC
            float w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = ok && k + j < k1 ? g.w[(long)(e0 + k + j) * g.v + c] : 0.f;
#pragma unroll
            for (int j = 0; j < 16; j += 4)
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const f32x4 xv = *(const f32x4*)(xs + i * RC + k + j);
#pragma unroll
                    for (int t = 0; t < 4; ++t) z[i] = __builtin_fmaf(w[j + t], xv[t], z[i]);
                }
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) red[(wv * RT + i) * 64 + lane] = z[i];
    __syncthreads();
    const float b = ok ? (g.b ? g.b[c] : 0.f) : -__builtin_inff();
    for (int i = wv; i < RT; i += 4) {
        const float all = (red[i * 64 + lane] + red[(RT + i) * 64 + lane]) + (red[(2 * RT + i) * 64 + lane] + red[(3 * RT + i) * 64 + lane]);
        const float s = masked(b) ? 0.f : all;
        const float t = (s + b) * kLog2e;
        zs[i * 64 + lane] = s + b >= kLowest ? fmaxf(t, kLowest) : t;
    }
}

template <int RT, bool XF32>
__global__ __launch_bounds__(256) void xent_rows_fwd_kernel(XentRows g) {
    __shared__ __attribute__((aligned(16))) float xs[RT * RC], red[4 * RT * 64], zs[RT * 64];
    xent_rows_logits<RT, XF32>(g, xs, red, zs);
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    for (int i = wv; i < g.n; i += 4) {             // the wave that wrote row i of zs
        const float z = zs[i * 64 + lane];
        float m = fmaxf(z, kLowest);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        float s = __builtin_amdgcn_exp2f(z - m);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
        if (lane == 0) g.part[(long)blockIdx.x * g.n + i] = make_float2(m, s);
        if ((long)blockIdx.x * 64 + lane == g.labels[i] && g.labels[i] < g.v) g.zlab[i] = z;
    }
}

// one row per workgroup of 64: its parts, a lane every 64th, then across the lanes
__global__ __launch_bounds__(64) void xent_rows_join_kernel(XentRows g, float* __restrict__ loss, float* __restrict__ lse,
                                                            int* __restrict__ hits, long parts) {
    const int i = blockIdx.x, lane = threadIdx.x;
    float m = kLowest, s = 0.f;
    auto join = [&](float pm, float ps) {
        const float mm = fmaxf(m, pm);
        s = s * __builtin_amdgcn_exp2f(m - mm) + ps * __builtin_amdgcn_exp2f(pm - mm);
        m = mm;
    };
    for (long p = lane; p < parts; p += 64) {
        const float2 q = g.part[p * g.n + i];
        join(q.x, q.y);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) join(__shfl_xor(m, off, 64), __shfl_xor(s, off, 64));
    if (lane == 0) {
        const int lab = g.labels[i];
        const bool ok = lab >= 0 && lab < g.v;
        const float z = ok ? g.zlab[i] : 0.f, ls = __builtin_amdgcn_logf(s);
        loss[i] = ok ? row_loss(m, ls, z, g.b ? g.b[lab] : 0.f) : 0.f;
        lse[i] = ok ? (m + ls) * kLn2 : 0.f;
        if (hits) hits[i] = ok && z >= m ? 1 : 0;
    }
}

template <int RT, bool XF32>
__global__ __launch_bounds__(256) void xent_rows_bwd_kernel(XentRows g) {
    __shared__ __attribute__((aligned(16))) float xs[RT * RC], red[4 * RT * 64], zs[RT * 64], wt[64][65];
    xent_rows_logits<RT, XF32>(g, xs, red, zs);
    float* dzt = red;                               // dz as [class][row], for reads of all rows of a class
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const long c = (long)blockIdx.x * 64 + lane;
    __syncthreads();
    for (int k = tid; k < RT * 64; k += 256) {      // zs becomes dz
        const int i = k >> 6;
        const int lab = i < g.n ? g.labels[i] : -1;
        float d = 0.f;
        if (lab >= 0 && lab < g.v) {
            const float p = __builtin_amdgcn_exp2f(zs[k] - lse_units(g.lse[i]));
            d = ((long)blockIdx.x * 64 + (k & 63) == lab ? p - 1.f : p) * g.dloss[i];
        }
        zs[k] = d;
        dzt[(k & 63) * RT + i] = d;
    }
    __syncthreads();
    const bool used = c < g.v && !(g.b && masked(g.b[c]));
    float dz[RT];                                   // of the lane's class
#pragma unroll
    for (int i = 0; i < RT; ++i) dz[i] = zs[i * 64 + lane];
    if (g.db && wv == 0 && c < g.v) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < RT; ++i) s += dz[i];
        g.db[c] = g.accumulate ? g.db[c] + s : s;
    }
    for (int e0 = 0; e0 < g.e; e0 += RC) {
        const int cnt = g.e - e0 < RC ? g.e - e0 : RC;
        if (g.e > RC) {                             // otherwise the stage of the logits is still there
            __syncthreads();
            xent_rows_stage<RT, XF32>(g, xs, e0, cnt);
            __syncthreads();
        }
        if (g.dw && c < g.v) {
            for (int k = 4 * wv; k < cnt; k += 16) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const f32x4 xv = *(const f32x4*)(xs + i * RC + k);
#pragma unroll
                    for (int t = 0; t < 4; ++t) s[t] = __builtin_fmaf(xv[t], dz[i], s[t]);
                }
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if (k + t < cnt) {
                        float* d = g.dw + (long)(e0 + k + t) * g.v + c;
                        *d = g.accumulate ? *d + s[t] : s[t];
                    }
                }
            }
        }
        if (g.dxp) {
            for (int k0 = 0; k0 < cnt; k0 += 64) {
                float w[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int k = k0 + wv + 4 * j;
                    w[j] = k < cnt && used ? g.w[(long)(e0 + k) * g.v + c] : 0.f;
                }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 16; ++j) wt[wv + 4 * j][lane] = w[j];
                __syncthreads();
                const int k = tid >> 2, q = tid & 3;
                float s[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i) s[i] = 0.f;
#pragma unroll 4
                for (int j = 0; j < 16; ++j) {
                    const float w1 = wt[k][4 * j + q];
#pragma unroll
                    for (int i = 0; i < RT; ++i) s[i] = __builtin_fmaf(w1, dzt[(4 * j + q) * RT + i], s[i]);
                }
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    s[i] += __shfl_xor(s[i], 1, 64);
                    s[i] += __shfl_xor(s[i], 2, 64);
                    if (q == 0 && i < g.n && k0 + k < cnt) g.dxp[((long)blockIdx.x * g.n + i) * g.e + e0 + k0 + k] = s[i];
                }
            }
        }
    }
}

// dx of 64 consecutive values per workgroup: 16 groups of parts, then the groups in order
__global__ __launch_bounds__(1024) void xent_rows_dx_kernel(const float* __restrict__ dxp, void* __restrict__ dx, int dx_f32, long total,
                                                            long parts) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
    const long i = (long)blockIdx.x * 64 + lane;
    float s = 0.f;
    if (i < total)
        for (long p = q; p < parts; p += 16) s += dxp[p * total + i];
    red[q][lane] = s;
    __syncthreads();
    if (q == 0 && i < total) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += red[k][lane];
        if (dx_f32) ((float*)dx)[i] = s;
        else ((bf16_t*)dx)[i] = (bf16_t)s;
    }
}

// ---------------------------------------------------------------- a block of rows
// Up to 128 rows (RB blocks of 32) W and dW are still what a call moves, but the products belong on the matrix pipe: float32
// instructions on W as it lies in memory, no powers of two and no planes.  A block of rows needs 64 cycles of a SIMD for every 64 values
// of W and product: with one block the four SIMDs of a CU would take 16 bytes of W a cycle, 8 TB/s over the chip.
//   logits: a workgroup takes 32 classes, its waves a quarter of the features each; W goes from memory to the A fragments (a lane a
//       class), x comes transposed from the cache.  Forward: (maximum, sum) per row; backward: dz (rows x classes) and db.
//   dx: 128 features a workgroup over a part of the classes, tiles of W and dz by LDS-DMA (a ring of three).
//   dW: a wave keeps dz of 32 classes and multiplies it with the features, 32 at a time.
struct XentShort {
    const void* x;
    const float *w, *b, *lse, *dloss;
    const int* labels;
    float *xt, *xz;                   // x with zeros for rows without a label, features x rows and rows x features
    float* bias;                      // classes padded with -inf
    float2* row;                      // lse in units of log 2 and dloss; (inf, 0) without a label
    int* lab;
    float2* part;                     // forward: (maximum, sum) per 32 classes and row
    float *zlab, *dz, *dxp, *dw, *db;
    long v, vp;                       // classes, padded to 128
    int n, e, ep, np, accumulate;     // features padded to 128, rows to 32
};

template <bool XF32>
__global__ __launch_bounds__(256) void xent_short_prep_kernel(XentShort g, int tiles) {
    __shared__ float t[64][33];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < tiles) {                    // 32 rows x 64 features
        const int rbs = g.np / 32, r0 = (int)blockIdx.x % rbs * 32, k0 = (int)blockIdx.x / rbs * 64, k = k0 + (tid & 63);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int rr = (tid >> 6) + 4 * i, row = r0 + rr;
            float a = 0.f;
            if (row < g.n && k < g.e) {
                const int lab = g.labels[row];
                const long at = (long)row * g.e + k;
                if (lab >= 0 && lab < g.v) a = XF32 ? ((const float*)g.x)[at] : (float)((const bf16_t*)g.x)[at];
            }
            if (g.xz) g.xz[(long)row * g.ep + k] = a;
            t[tid & 63][rr] = a;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int kk = (tid >> 5) + 8 * i;
            g.xt[(long)(k0 + kk) * g.np + r0 + (tid & 31)] = t[kk][tid & 31];
        }
    } else {
        const long first = (long)(blockIdx.x - tiles) * 256 + tid, stride = (long)(gridDim.x - tiles) * 256;
        for (long c = first; c < g.vp; c += stride) g.bias[c] = c < g.v ? (g.b ? g.b[c] : 0.f) : -__builtin_inff();
        for (long i = first; i < g.np; i += stride) {
            int lab = i < g.n ? g.labels[i] : -1;
            if (lab < 0 || lab >= g.v) lab = -1;
            g.lab[i] = lab;
            if (g.row) g.row[i] = lab < 0 ? make_float2(__builtin_inff(), 0.f) : make_float2(lse_units(g.lse[i]), g.dloss[i]);
        }
    }
}

template <int RB, bool BWD>
__global__ __launch_bounds__(256) void xent_short_logits_kernel(XentShort g) {
    __shared__ float red[4 * 16 * 64], zs[32 * RB * 33];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = lane & 31, h = lane >> 5;
    const long c0 = (long)blockIdx.x * 32, c = c0 + r < g.v ? c0 + r : g.v - 1;
    const int span = (g.e + 63) / 64 * 16, kb = wv * span, end = (g.e + 15) / 16 * 16, ke = kb + span < end ? kb + span : end;
    f32x16 acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] = 0.f;
    // 16 features: the lane's class and row, features k + h, k + h + 2, ...
    auto fetch = [&](int k, float (&a)[8], float (&x)[RB][8]) {
        const float* wp = g.w + (long)(k + h) * g.v + c;
        if (k + 16 <= g.e) {
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = wp[2 * j * g.v];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = k + 2 * j + h < g.e ? wp[2 * j * g.v] : 0.f;
        }
        const float* xp = g.xt + (long)(k + h) * g.np + r;
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[b][j] = xp[2 * j * g.np + 32 * b];
    };
    auto products = [&](const float (&a)[8], const float (&x)[RB][8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int b = 0; b < RB; ++b) acc[b] = mfma32(a[j], x[b][j], acc[b]);
    };
    if (kb < ke) {
        float a0[8], a1[8], x0[RB][8], x1[RB][8];
        fetch(kb, a0, x0);
        for (int k = kb; k < ke; k += 32) {
            if (k + 16 < ke) fetch(k + 16, a1, x1);
            products(a0, x0);
            if (k + 16 < ke) {
                if (k + 32 < ke) fetch(k + 32, a0, x0);
                products(a1, x1);
            }
        }
    }
    // the waves' sums in order; wave wv finishes the classes 8 wv + 4 h + {0 .. 3}
    float bv[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) bv[t] = g.bias[c0 + 8 * wv + 4 * h + t];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) red[(wv * 16 + i) * 64 + lane] = acc[b][i];
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const float* q = red + (4 * wv + t) * 64 + lane;
            const float all = (q[0] + q[16 * 64]) + (q[32 * 64] + q[48 * 64]);
            const float z = (masked(bv[t]) ? 0.f : all) + bv[t], u = z * kLog2e;
            zs[(32 * b + r) * 33 + 8 * wv + 4 * h + t] = z >= kLowest ? fmaxf(u, kLowest) : u;
        }
        __syncthreads();
    }
    const int q = tid & 7;                              // eight lanes a row, four classes each
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int row = 32 * b + (tid >> 3);
        const long rel = g.lab[row] - c0;               // the label's place, if it is one of the 32
        float* zr = zs + row * 33 + 4 * q;
        if constexpr (!BWD) {
            float m = kLowest, s = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = fmaxf(m, zr[i]);
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
#pragma unroll
            for (int i = 0; i < 4; ++i) s += __builtin_amdgcn_exp2f(zr[i] - m);
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) s += __shfl_xor(s, off, 64);
            if (q == 0) g.part[(long)row * gridDim.x + blockIdx.x] = make_float2(m, s);
            if (rel >= 4 * q && rel < 4 * q + 4 && g.lab[row] >= 0) g.zlab[row] = zr[rel - 4 * q];
        } else {
            const float2 info = g.row[row];
            f32x4 d;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(zr[i] - info.x);
                d[i] = (g.lab[row] >= 0 && rel == 4 * q + i ? p - 1.f : p) * info.y;
                zr[i] = d[i];
            }
            *(f32x4*)(g.dz + (long)row * g.vp + c0 + 4 * q) = d;
        }
    }
    if (BWD && g.db) {
        const int cl = tid & 31, part = tid >> 5;
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * RB; ++i) s += zs[(part * 4 * RB + i) * 33 + cl];
        red[part * 32 + cl] = s;
        __syncthreads();
        if (tid < 32 && c0 + cl < g.v) {
            s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += red[i * 32 + cl];
            g.db[c0 + cl] = g.accumulate ? g.db[c0 + cl] + s : s;
        }
    }
}

// The same for many classes: a workgroup takes 128 of them (a wave 32) and walks the features 32 at a time, tiles of W and of x by
// LDS-DMA (a ring of three), so that x is read a quarter as often.  W16: rows of W consist of 16-byte pieces.
template <int RB, bool BWD, bool W16>
__global__ __launch_bounds__(256) void xent_short_tiled_kernel(XentShort g) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    constexpr int WB = 32 * 512, XB = RB * 4096, BUF = WB + XB, PIECES = (W16 ? 4 : 16) + RB;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
    const long c0 = (long)blockIdx.x * 128;
    const int steps = (g.e + 31) / 32;
    // step it; features past the last meet zeros of x, classes past the last are the last ones and get their own place masked
    auto stage = [&](int it) {
        const unsigned dst = lds_byte(lds) + it % 3 * BUF;
        constexpr int PER = W16 ? 4 : 16;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int piece = wv * PER + i;
            if constexpr (W16) {                          // 2 rows of 512 B
                const int k = it * 32 + piece * 2, ka = k < g.e ? k : g.e - 1, kr = k + h < g.e ? k + h : g.e - 1;
                const long c = c0 + 4 * r < g.v ? 4 * r : g.v - 4 - c0;
                lds_dma16(g.w + ka * g.v + c0, (int)(((kr - ka) * g.v + c) * 4), dst + piece * 1024);
            } else {                                      // half a row
                const int k = it * 32 + piece / 2, ka = k < g.e ? k : g.e - 1, cl = piece % 2 * 64 + lane;
                const long c = c0 + cl < g.v ? cl : g.v - 1 - c0;
                lds_dma4(g.w + ka * g.v + c0, (int)(c * 4), dst + piece * 256);
            }
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {                    // 32 features x np rows as they lie in xt
            const int piece = wv * RB + i;
            lds_dma16(g.xt + (long)it * 32 * g.np + piece * 256, lane * 16, dst + WB + piece * 1024);
        }
    };
    f32x16 acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] = 0.f;
    stage(0);
    if (steps > 1) stage(1);
    for (int it = 0; it < steps; ++it) {
        if (it + 1 < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (it + 2 < steps) stage(it + 2);
        const unsigned char* buf = lds + it % 3 * BUF;
        const float *wt = (const float*)buf + h * 128 + 32 * wv + r, *xt = (const float*)(buf + WB) + h * 32 * RB + r;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float a = wt[2 * j * 128];
#pragma unroll
            for (int b = 0; b < RB; ++b) acc[b] = mfma32(a, xt[2 * j * 32 * RB + 32 * b], acc[b]);
        }
    }
    // lane: row 32 b + r, classes 8 q + 4 h + {0 .. 3} of the wave's
    const long cw = c0 + 32 * wv;
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 bv = *(const f32x4*)(g.bias + cw + 8 * q + 4 * h);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float z = (masked(bv[k]) ? 0.f : acc[b][4 * q + k]) + bv[k], u = z * kLog2e;
                acc[b][4 * q + k] = z >= kLowest ? fmaxf(u, kLowest) : u;
            }
        }
    float db[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) db[i] = 0.f;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int row = 32 * b + r, lab = g.lab[row];
        const long rel = lab < 0 ? -1 : lab - cw - 4 * h;
        if constexpr (!BWD) {
            float m = kLowest, s = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, acc[b][i]);
            m = fmaxf(m, __shfl_xor(m, 32, 64));
#pragma unroll
            for (int i = 0; i < 16; ++i) s += __builtin_amdgcn_exp2f(acc[b][i] - m);
            s += __shfl_xor(s, 32, 64);
            if (h == 0) g.part[((long)row * gridDim.x + blockIdx.x) * 4 + wv] = make_float2(m, s);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (rel == (i & 3) + 8 * (i >> 2)) g.zlab[row] = acc[b][i];
        } else {
            const float2 info = g.row[row];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 d;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float p = __builtin_amdgcn_exp2f(acc[b][4 * q + k] - info.x);
                    d[k] = (rel == 8 * q + k ? p - 1.f : p) * info.y;
                    db[4 * q + k] += d[k];
                }
                *(f32x4*)(g.dz + (long)row * g.vp + cw + 8 * q + 4 * h) = d;
            }
        }
    }
    if (BWD && g.db) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) db[i] += __shfl_xor(db[i], off, 64);
            const long c = cw + acc_row(i, lane);
            if (r == i && c < g.v) g.db[c] = g.accumulate ? g.db[c] + db[i] : db[i];
        }
    }
}

// loss and lse of a row: a thread every 256th part, then across the threads
__global__ __launch_bounds__(256) void xent_short_join_kernel(XentShort g, float* __restrict__ loss, float* __restrict__ lse,
                                                              int* __restrict__ hits, int parts) {
    __shared__ float2 red[4];
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    float m = kLowest, s = 0.f;
    auto join = [&](float pm, float ps) {
        const float mm = fmaxf(m, pm);
        s = s * __builtin_amdgcn_exp2f(m - mm) + ps * __builtin_amdgcn_exp2f(pm - mm);
        m = mm;
    };
    for (int p = threadIdx.x; p < parts; p += 1024) {           // four loads in flight
        float2 q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = p + 256 * k < parts ? g.part[(long)row * parts + p + 256 * k] : make_float2(kLowest, 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) join(q[k].x, q[k].y);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float pm = __shfl_xor(m, off, 64), ps = __shfl_xor(s, off, 64);
        join(pm, ps);
    }
    if (lane == 0) red[threadIdx.x >> 6] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 4; ++k) join(red[k].x, red[k].y);
        const int lab = g.lab[row];
        const float z = lab >= 0 ? g.zlab[row] : 0.f, ls = __builtin_amdgcn_logf(s);
        loss[row] = lab >= 0 ? row_loss(m, ls, z, g.b ? g.b[lab] : 0.f) : 0.f;
        lse[row] = lab >= 0 ? (m + ls) * kLn2 : 0.f;
        if (hits) hits[row] = lab >= 0 && z >= m ? 1 : 0;
    }
}

// W16: rows of W consist of 16-byte pieces.  Staged rows are 32 classes (128 B); 16-byte chunks are XOR-swizzled by the row so that
// the 16 rows of a read cover all banks.
template <int RB, bool W16>
__global__ __launch_bounds__(256) void xent_short_dx_kernel(XentShort g) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    constexpr int WB = 128 * 128, DB = RB * 4096, BUF = WB + DB + 128, PIECES = (W16 ? 4 : 16) + RB + 1;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
    const int k0 = blockIdx.x * 128, tiles = (int)((g.v + 31) / 32), per = (tiles + gridDim.y - 1) / gridDim.y;
    const int t0 = blockIdx.y * per, t1 = t0 + per < tiles ? t0 + per : tiles;
    // tile t: features past the last and classes past the last are those themselves; the former are not stored, the latter masked
    auto stage = [&](int t) {
        const unsigned dst = lds_byte(lds) + (t - t0) % 3 * BUF;
        const long c0 = (long)t * 32;
        constexpr int ROWS = W16 ? 8 : 2, PER = W16 ? 4 : 16;          // rows of an instruction, instructions of a wave
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int piece = wv * PER + i, row = piece * ROWS + lane / (64 / ROWS);
            const int kf = k0 + piece * ROWS < g.e ? k0 + piece * ROWS : g.e - 1, kr = k0 + row < g.e ? k0 + row : g.e - 1;
            const int s = (row >> 1) & 7;
            long c = W16 ? c0 + 4 * ((lane & 7) ^ s) : c0 + 4 * (((lane & 31) >> 2) ^ s) + (lane & 3);
            c = c < g.v ? c : g.v - (W16 ? 4 : 1);
            const int off = (int)(((kr - kf) * g.v + c - c0) * 4);
            if constexpr (W16) lds_dma16(g.w + kf * g.v + c0, off, dst + piece * 1024);
            else lds_dma4(g.w + kf * g.v + c0, off, dst + piece * 256);
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            const int piece = wv * RB + i, row = lane >> 3;
            const int off = (int)(row * g.vp * 4) + (((lane & 7) ^ (((piece * 8 + row) >> 1) & 7)) << 4);
            lds_dma16(g.dz + piece * 8 * g.vp + c0, off, dst + WB + piece * 1024);
        }
        if (lane < 32) lds_dma4(g.bias + c0, lane * 4, dst + WB + DB);      // every wave the same: each counts its own loads only
    };
    f32x16 acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] = 0.f;
    if (t0 < t1) stage(t0);
    if (t0 + 1 < t1) stage(t0 + 1);
    const int sw = (r >> 1) & 7;
    for (int t = t0; t < t1; ++t) {
        if (t + 1 < t1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (t + 2 < t1) stage(t + 2);
        const unsigned char* buf = lds + (t - t0) % 3 * BUF;
#pragma unroll
        for (int q = 0; q < 4; ++q) {                   // classes 8 q + 4 h + {0 .. 3}
            const int at = ((2 * q + h) ^ sw) << 4;
            const f32x4 bias = *(const f32x4*)(buf + WB + DB + (8 * q + 4 * h) * 4);
            f32x4 a = *(const f32x4*)(buf + (32 * wv + r) * 128 + at), d[RB];
#pragma unroll
            for (int b = 0; b < RB; ++b) d[b] = *(const f32x4*)(buf + WB + (32 * b + r) * 128 + at);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w = masked(bias[j]) ? 0.f : a[j];
#pragma unroll
                for (int b = 0; b < RB; ++b) acc[b] = mfma32(w, d[b][j], acc[b]);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        float* o = g.dxp + ((long)blockIdx.y * g.np + 32 * b + r) * g.ep + k0 + 32 * wv + 4 * h;
#pragma unroll
        for (int q = 0; q < 4; ++q) *(f32x4*)(o + 8 * q) = (f32x4){acc[b][4 * q], acc[b][4 * q + 1], acc[b][4 * q + 2], acc[b][4 * q + 3]};
    }
}

// kg blocks of 32 features a workgroup.  The stores of a step are never skipped (an offset past the end of the buffer drops them), so
// that a wait can count them: behind the DMA of a step come the stores of two steps and the DMA of one.
template <int RB>
__global__ __launch_bounds__(256) void xent_short_dw_kernel(XentShort g, int kg) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    constexpr int BUF = RB * 4096;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
    const long c = (long)blockIdx.x * 128 + wv * 32 + r;
    const int blocks = (g.e + 31) / 32, t0 = blockIdx.y * kg, t1 = t0 + kg < blocks ? t0 + kg : blocks;
    auto stage = [&](int t) {                            // np rows x 32 features
        const unsigned dst = lds_byte(lds) + (t - t0) % 3 * BUF;
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            const int piece = wv * RB + i;               // 8 rows of 128 B
            lds_dma16(g.xz + (long)piece * 8 * g.ep + t * 32, ((lane >> 3) * g.ep + (lane & 7) * 4) * 4, dst + piece * 1024);
        }
    };
    float d[16 * RB];
#pragma unroll
    for (int j = 0; j < 16 * RB; ++j) d[j] = g.dz[(2 * j + h) * g.vp + c];
#pragma unroll
    for (int j = 0; j < 16 * RB; ++j) asm volatile("" : "+v"(d[j]));          // here already: or every step waits for them by count
    stage(t0);
    if (t0 + 1 < t1) stage(t0 + 1);
    for (int t = t0; t < t1; ++t) {
        if (t + 1 >= t1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else if (t < t0 + 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(RB) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(RB + 32) : "memory");
        __syncthreads();
        if (t + 2 < t1) stage(t + 2);
        const float* xt = (const float*)(lds + (t - t0) % 3 * BUF) + h * 32 + r;
        f32x16 acc;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 16 * RB; ++j) acc = mfma32(xt[2 * j * 32], d[j], acc);
        float* rows = g.dw + (long)t * 32 * g.v;
        const int left = g.e - t * 32 < 32 ? g.e - t * 32 : 32;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(rows, 0, (unsigned)(left * g.v * 4), 0x00020000);
        auto at = [&](int i) { return c < g.v ? (unsigned)(acc_row(i, lane) * g.v + c) * 4u : 0xfffffff0u; };
        float old[16];
        if (g.accumulate) {
#pragma unroll
            for (int i = 0; i < 16; ++i) old[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, at(i), 0, 0));
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] += old[i];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float q = acc[i];
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, q), rs, at(i), 0, 0);
        }
    }
}

__global__ __launch_bounds__(256) void xent_zero_kernel(float* __restrict__ a, long na, float* __restrict__ b, long nb) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < na || i < nb; i += (long)gridDim.x * 256) {
        if (i < na) a[i] = 0.f;
        if (i < nb) b[i] = 0.f;
    }
}

// ---------------------------------------------------------------- host
template <bool XF32>
int few_forward(const XentRows& g, float* loss, float* lse, int* hits, hipStream_t st) {
    const dim3 grid((unsigned)(up(g.v, 64) / 64)), block(256);
    if (g.n == 1) hipLaunchKernelGGL((xent_rows_fwd_kernel<1, XF32>), grid, block, 0, st, g);
    else if (g.n <= 4) hipLaunchKernelGGL((xent_rows_fwd_kernel<4, XF32>), grid, block, 0, st, g);
    else hipLaunchKernelGGL((xent_rows_fwd_kernel<16, XF32>), grid, block, 0, st, g);
    hipLaunchKernelGGL(xent_rows_join_kernel, dim3((unsigned)g.n), dim3(64), 0, st, g, loss, lse, hits, (long)grid.x);
    return mgx_launch_status();
}

template <bool XF32>
int few_backward(const XentRows& g, void* dx, hipStream_t st) {
    const dim3 grid((unsigned)(up(g.v, 64) / 64)), block(256);
    if (g.n == 1) hipLaunchKernelGGL((xent_rows_bwd_kernel<1, XF32>), grid, block, 0, st, g);
    else if (g.n <= 4) hipLaunchKernelGGL((xent_rows_bwd_kernel<4, XF32>), grid, block, 0, st, g);
    else hipLaunchKernelGGL((xent_rows_bwd_kernel<16, XF32>), grid, block, 0, st, g);
    const long total = (long)g.n * g.e;
    if (dx)
        hipLaunchKernelGGL(xent_rows_dx_kernel, dim3((unsigned)(up(total, 64) / 64)), dim3(1024), 0, st, g.dxp, dx, (int)XF32, total,
                           (long)grid.x);
    return mgx_launch_status();
}

// workspace of the few-rows form: parts and label logits, or the parts of dx
int64_t few_bytes(int64_t n, int64_t e, int64_t v, bool backward) {
    const int64_t parts = up(v, 64) / 64;
    return backward ? parts * n * e * 4 : up(parts * n * 8, 16) + n * 4;
}

struct Layout {
    bool narrow;                   // the streamed kernels
    int rows_wg;                   // resident rows of a workgroup (FWD, DX)
    int64_t np, vp, ep, vc, nz, nf, nx;      // nf, nx, nz: parts of the streamed operand in FWD, DX, DW (nz: of the rows in general)
    int64_t vm;                    // classes of a piece whose dW is not split, before the ones whose dW has nz parts
    int64_t part, bias, exps, rmax, lab, zlab, row, ones, xh, xl, xsh, xsl, wh, wl, slices, dzh, dzl, dxw, slabs, slabs_b, total;
};

Layout layout(int64_t n, int64_t e, int64_t v, bool xf32, bool backward) {
    Layout l = {};
    l.narrow = e <= 128;
    l.rows_wg = l.narrow && xf32 ? 128 : 256;
    l.np = up(n, l.rows_wg);
    l.vp = up(v, l.narrow ? 128 : 256);
    l.ep = e <= 64 ? 64 : up(e, 128);
    // Parts of a contraction of `tiles` steps by `wgs` workgroups, `slots` of which run at once: a step takes step_us, and each part
    // costs a start of half a step's latency (1 us) and `bytes` written and read once more for the join at 4 TB/s (one part
    // of dW goes to the gradient itself).  Swept over the parts, the choice was within 5 % of the best from 300 x 64 x 3001
    // to 700 x 128 x 65536 and 8000 x 100 x 1500.
    auto split = [](int64_t wgs, int64_t tiles, int64_t slots, double step_us, double bytes, bool direct = false, double* time = nullptr) {
        int64_t best = 1;
        double least = 1e30;
        for (int64_t p = 1; p <= 128 && (p == 1 || tiles / p >= 4); ++p) {
            const double rounds = (double)((wgs * p + slots - 1) / slots);
            const double join = direct && p == 1 ? 0.0 : 4.0 + (double)p * (bytes * 2.0 / 4e6 + 0.05);
            const double t = rounds * ((double)((tiles + p - 1) / p) * step_us + 1.0) + join;
            if (t < least) {
                least = t;
                best = p;
            }
        }
        if (time) *time = least;
        return best;
    };
    if (l.narrow) {      // step times: 128 (256) resident items x 32 streamed x 128 (64) features at 1 PFLOP/s over the slots
        const double f = l.ep == 64 ? 0.6 : 1.0;
        l.nf = split(l.np / l.rows_wg, l.vp / ST, 512, f * (xf32 ? 1.6 : 2.1), 8.0 * (double)l.np);
        l.nx = split(l.np / l.rows_wg, l.vp / ST, xf32 || l.ep == 64 ? 512 : 256, f * (xf32 ? 3.2 : l.ep == 64 ? 3.3 : 1.65),
                     4.0 * (double)(l.np * l.ep));
        l.nz = split(l.vp / 128, l.np / ST, 512, f * (xf32 ? 3.2 : 2.1), 4.0 * (double)(l.ep * l.vp), true);
    }
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += up(bytes, 1024);
        return o;
    };
    l.part = take(3 * kMaxParts * 4);
    l.exps = take(16);
    l.rmax = take(l.np * 4);
    l.row = take(l.np * 16);
    l.bias = take(l.vp * 4);
    l.lab = take(l.np * 4);
    l.xh = take(l.np * l.ep * 2);
    l.xl = xf32 ? take(l.np * l.ep * 2) : 0;
    l.wh = take(l.vp * l.ep * 2);
    l.wl = take(l.vp * l.ep * 2);
    if (!backward) {
        l.zlab = take(l.np * 4);
        if (!l.narrow) l.nf = l.vp / 64;
        l.slices = take(l.np * l.nf * 8);
    } else if (l.narrow) {
        l.vc = l.vp;
        l.dxw = take(l.nx * l.np * l.ep * 4);
        l.slabs = l.nz > 1 ? take(l.nz * l.ep * l.vp * 4) : 0;
        l.slabs_b = l.nz > 1 ? take(l.nz * l.vp * 4) : 0;
    } else {
        l.ones = take(l.np * 2);
        l.xsh = take(l.np * l.ep * 2);
        l.xsl = xf32 ? take(l.np * l.ep * 2) : 0;
        // a piece of the classes: dz planes of about 128 MB, which the 256 MB last-level cache holds
        l.vc = (int64_t)(128 << 20) / (4 * l.np) / 256 * 256;
        if (l.vc < 256) l.vc = 256;
        if (l.vc > l.vp) l.vc = l.vp;
        // a step: 256 x 128 x 32 with one to three plane products at 1 PFLOP/s over the slots
        l.nx = split((l.np / 256) * (l.ep / 128), l.vc / BK, 256, xf32 ? 1.6 : 0.55, 4.0 * (double)(l.np * l.ep));
        // dW: the classes of a piece that fill whole rounds of the 256 CUs are not split, a part round behind them is
        // (1501 x 1000 x 10001 float32, 320 tiles: dW and its join 127 us, 155 us as two rounds)
        const double step = xf32 ? 1.6 : 1.1;
        const int64_t gx = l.ep / 128, gy = l.vc / 256, gm = gx * gy / 256 * 256 / gx;
        double whole, tail = 0.0;
        l.nz = split(gx * gy, l.np / BK, 256, step, 4.0 * (double)(l.ep * l.vc), true, &whole);
        if (gm > 0 && gm < gy) {
            const int64_t nt = split(gx * (gy - gm), l.np / BK, 256, step, 4.0 * (double)(l.ep * 256 * (gy - gm)), true, &tail);
            const double rounds = (double)((gx * gm + 255) / 256);
            if (rounds * ((double)(l.np / BK) * step + 1.0) + 3.0 + tail < whole) {
                l.nz = nt;
                l.vm = 256 * gm;
            }
        }
        const int64_t vs = l.vc - l.vm;
        l.dzh = take(l.np * l.vc * 2);
        l.dzl = take(l.np * l.vc * 2);
        l.dxw = take(l.nx * l.np * l.ep * 4);
        l.slabs = l.nz > 1 ? take(l.nz * l.ep * vs * 4) : 0;
        l.slabs_b = l.nz > 1 ? take(l.nz * vs * 4) : 0;
    }
    l.total = at;
    return l;
}

bool sizes_ok(int64_t n, int64_t e, int64_t v) {
    return n >= 0 && e >= 1 && v >= 1 && n <= 8000000 && v <= 8000000 && e <= 65000;      // rows / 128, classes / 128 and e + 1 are grid dimensions
}

// m x n results in `parts` parts of the contraction; WM waves of 64 along m, 8 / WM along n
template <int NA, int NB, bool AT, bool BT, int EPI, int WM>
void launch_gemm(const XentGemm& g, int64_t m, int64_t n, int64_t parts, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    constexpr int bytes = 3 * (NA * 64 * WM + NB * 512 / WM) * BK * 2 + (EPI == EPI_DW ? 3 * 64 : 0);
    mgx_allow_dynamic_lds(xent_gemm_kernel<NA, NB, AT, BT, EPI, WM>, bytes, done);
    hipLaunchKernelGGL((xent_gemm_kernel<NA, NB, AT, BT, EPI, WM>), dim3((unsigned)(m / (64 * WM)), (unsigned)(n / (512 / WM)), (unsigned)parts),
                       dim3(512), bytes, st, g);
}

template <int EP, int NR, int NS, int RB, int MODE, int OCC>
void launch_stream_ep(const XentStream& g, int64_t wgs, int64_t parts, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    constexpr int bytes = 4 * (NS * ST * EP * 2 + 1024);
    mgx_allow_dynamic_lds(xent_stream_kernel<EP, NR, NS, RB, MODE, OCC>, bytes, done);
    hipLaunchKernelGGL((xent_stream_kernel<EP, NR, NS, RB, MODE, OCC>), dim3((unsigned)wgs, (unsigned)parts), dim3(256), bytes, st, g);
}

template <int NR, int NS, int RB, int MODE, int OCC>
void launch_stream(const Layout& l, const XentStream& g, int64_t wgs, int64_t parts, hipStream_t st) {
    if (l.ep == 64) launch_stream_ep<64, NR, NS, RB, MODE, 2>(g, wgs, parts, st);
    else launch_stream_ep<128, NR, NS, RB, MODE, OCC>(g, wgs, parts, st);
}

void launch_prep(const Layout& l, char* ws, const void* x, bool xf32, const float* w, const float* b, const int* labels,
                 const float* lse, const float* dloss, int64_t n, int64_t e, int64_t v, hipStream_t st) {
    int64_t parts = up(e * v / 16 + n * e / 16, 256) / 256;         // sixteen values a thread, up to four workgroups a CU
    parts = parts < 64 ? 64 : (parts > kMaxParts ? kMaxParts : parts);
    unsigned* part = (unsigned*)(ws + l.part);
    const bool vec = e % (xf32 ? 4 : 8) == 0;
    const int64_t cols = vec ? e / (xf32 ? 4 : 8) : e;
    int lsh = 0;                                                    // lanes of a row: up to 64, few enough for four loads each
    while (lsh < 6 && (4 << lsh) < cols) ++lsh;
    auto largest = [&](auto f32_, auto vec_, auto wvec_) {
        hipLaunchKernelGGL((xent_max_kernel<decltype(f32_)::value, decltype(vec_)::value, decltype(wvec_)::value>), dim3((unsigned)parts),
                           dim3(256), 0, st, w, b, x, (long)n, (int)e, labels, (long)v, lsh, dloss, part, (unsigned*)(ws + l.rmax));
    };
    const std::true_type yes;
    const std::false_type no;
    auto by_w = [&](auto f32_, auto vec_) { v % 4 == 0 ? largest(f32_, vec_, yes) : largest(f32_, vec_, no); };
    if (xf32) vec ? by_w(yes, yes) : by_w(yes, no);
    else vec ? by_w(no, yes) : by_w(no, no);
    XentPrep p = {};
    p.x = x; p.w = w; p.b = b; p.lse = lse; p.dloss = dloss; p.labels = labels; p.part = part; p.parts = (int)parts;
    p.n = n; p.v = v; p.np = l.np; p.vp = l.vp; p.e = (int)e; p.ep = (int)l.ep;
    p.xh = (f16_t*)(ws + l.xh); p.xl = (f16_t*)(ws + l.xl); p.wh = (f16_t*)(ws + l.wh); p.wl = (f16_t*)(ws + l.wl);
    p.bias = (float*)(ws + l.bias); p.exps = (int*)(ws + l.exps); p.rmax = (unsigned*)(ws + l.rmax); p.lab = (int*)(ws + l.lab);
    p.row = (f32x4*)(ws + l.row);
    if (dloss && !l.narrow) {
        p.ones = (f16_t*)(ws + l.ones); p.xsh = (f16_t*)(ws + l.xsh); p.xsl = (f16_t*)(ws + l.xsl);
    }
    p.wtiles = (l.vp / 64) * (l.ep / 64);
    p.xblocks = up(l.np * l.ep / 8, 256) / 256;
    if (p.xblocks > 2048) p.xblocks = 2048;
    const dim3 grid((unsigned)(p.wtiles + p.xblocks + 64));
    if (xf32) hipLaunchKernelGGL(xent_prep_kernel<true>, grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL(xent_prep_kernel<false>, grid, dim3(256), 0, st, p);
}

// dx from its parts (exps NULL: they are dx itself, not of the streamed or the wide products' planes), together with dW from its slabs
// where both remain to be done
void launch_joins(const XentDxJoin* j, const XentDwReduce* g, hipStream_t st) {
    // sixteen groups of parts: 200 x 128 x 65536 94.0 us a backward against 99.2 with one, 53 x 75 x 25145 52.5 against 57.8; with the
    // outputs of 3000 x 32 x 8192 one group fills the chip (67.9 against 77.7)
    const int64_t outs = j ? j->n * j->ep : 0;
    const bool groups = j && j->np >= 16 && outs <= 1 << 16;
    if (groups) hipLaunchKernelGGL(xent_dx_join_kernel<16>, dim3((unsigned)(up(outs, 64) / 64)), dim3(1024), 0, st, *j);
    int64_t blocks = up(outs, 256) / 256;
    blocks = blocks < 4096 ? blocks : 4096;
    if (g && j && !groups)
        hipLaunchKernelGGL(xent_joins_kernel, dim3((unsigned)(blocks + g->blocks())), dim3(256), 0, st, *j, (long)blocks, *g);
    else if (g) hipLaunchKernelGGL(xent_dw_reduce_kernel, dim3((unsigned)g->blocks()), dim3(256), 0, st, *g);
    else if (!groups) hipLaunchKernelGGL(xent_dx_join_kernel<1>, dim3((unsigned)blocks), dim3(256), 0, st, *j);
}

// ------------------------------------------------ a block of rows
struct ShortLayout {
    int64_t np, ep, vp, parts;
    int64_t lab, row, bias, xt, xz, part, zlab, dz, dxp, total;
};

ShortLayout short_layout(int64_t n, int64_t e, int64_t v, bool backward) {
    ShortLayout l = {};
    l.np = up(n, 32);
    l.ep = up(e, 128);
    l.vp = up(v, 128);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += up(bytes, 1024);
        return o;
    };
    l.lab = take(l.np * 4);
    l.bias = take(l.vp * 4);
    l.xt = take(l.ep * l.np * 4);
    if (backward) {
        l.row = take(l.np * 8);
        l.xz = take(l.ep * l.np * 4);
        l.dz = take(l.np * l.vp * 4);
        // dx: two workgroups a CU, eight tiles of classes each at least
        const int64_t wgs = l.ep / 128, tiles = up(v, 32) / 32;
        l.parts = 512 / wgs < tiles / 8 ? 512 / wgs : tiles / 8;
        if (l.parts < 1) l.parts = 1;
        l.dxp = take(l.parts * l.np * l.ep * 4);
    } else {
        l.part = take(up(v, 128) / 32 * l.np * 8);
        l.zlab = take(l.np * 4);
    }
    l.total = at;
    return l;
}

// Logits by tiles of 128 classes where these fill the chip, otherwise 32 classes a workgroup (forward + backward of 64 rows and 1000
// features: 59 + 156 us at 32768 classes, 81 + 168 the other way; 58 + 118 at 16384, 44 + 98 the other way).
inline bool short_tiled(int64_t v) { return v >= 32768; }
inline int64_t short_slices(int64_t v) { return short_tiled(v) ? up(v, 128) / 32 : up(v, 32) / 32; }

template <int RB, bool BWD, bool W16>
void launch_short_tiled(const XentShort& g, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    constexpr int bytes = 3 * (32 * 512 + RB * 4096);
    mgx_allow_dynamic_lds(xent_short_tiled_kernel<RB, BWD, W16>, bytes, done);
    hipLaunchKernelGGL((xent_short_tiled_kernel<RB, BWD, W16>), dim3((unsigned)(up(g.v, 128) / 128)), dim3(256), bytes, st, g);
}

template <int RB, bool BWD>
void launch_short_logits(const XentShort& g, hipStream_t st) {
    if (!short_tiled(g.v))
        hipLaunchKernelGGL((xent_short_logits_kernel<RB, BWD>), dim3((unsigned)(up(g.v, 32) / 32)), dim3(256), 0, st, g);
    else if (g.v % 4 == 0) launch_short_tiled<RB, BWD, true>(g, st);
    else launch_short_tiled<RB, BWD, false>(g, st);
}

template <int RB, bool W16>
void launch_short_dx(const XentShort& g, int64_t parts, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    constexpr int bytes = 3 * (128 * 128 + RB * 4096 + 128);
    mgx_allow_dynamic_lds(xent_short_dx_kernel<RB, W16>, bytes, done);
    hipLaunchKernelGGL((xent_short_dx_kernel<RB, W16>), dim3((unsigned)(g.ep / 128), (unsigned)parts), dim3(256), bytes, st, g);
}

template <int RB>
void short_backward(const XentShort& g, void* dx, bool xf32, int64_t parts, hipStream_t st) {
    launch_short_logits<RB, true>(g, st);
    if (dx) {
        if (g.v % 4 == 0) launch_short_dx<RB, true>(g, parts, st);
        else launch_short_dx<RB, false>(g, parts, st);
        const XentDxJoin j = {g.dxp, nullptr, nullptr, false, dx, (int)xf32, (int)parts, (long)g.np * g.ep, (long)g.n, g.e, g.ep};
        launch_joins(&j, nullptr, st);
    }
    if (g.dw) {
        const int64_t cols = up(g.v, 128) / 128, blocks = up(g.e, 32) / 32;
        int64_t kg = cols * blocks / 1024;               // four workgroups a CU where there is enough, up to 16 blocks each
        kg = kg < 1 ? 1 : (kg > 16 ? 16 : kg);
        hipLaunchKernelGGL(xent_short_dw_kernel<RB>, dim3((unsigned)cols, (unsigned)(up(blocks, kg) / kg)), dim3(256), 3 * RB * 4096, st, g, (int)kg);
    }
}

int short_call(XentShort g, bool xf32, const ShortLayout& l, char* ws, float* loss, float* lse, int* hits, void* dx, bool backward,
               hipStream_t st) {
    g.np = (int)l.np; g.ep = (int)l.ep; g.vp = l.vp;
    g.lab = (int*)(ws + l.lab); g.bias = (float*)(ws + l.bias); g.xt = (float*)(ws + l.xt);
    if (backward) {
        g.row = (float2*)(ws + l.row); g.xz = (float*)(ws + l.xz); g.dz = (float*)(ws + l.dz); g.dxp = (float*)(ws + l.dxp);
    } else {
        g.part = (float2*)(ws + l.part); g.zlab = (float*)(ws + l.zlab);
    }
    const int tiles = (int)(l.np / 32 * (l.ep / 64));
    const dim3 grid((unsigned)(tiles + 64));
    if (xf32) hipLaunchKernelGGL(xent_short_prep_kernel<true>, grid, dim3(256), 0, st, g, tiles);
    else hipLaunchKernelGGL(xent_short_prep_kernel<false>, grid, dim3(256), 0, st, g, tiles);
    const int rb = g.np / 32;
    if (backward) {
        if (rb == 1) short_backward<1>(g, dx, xf32, l.parts, st);
        else if (rb == 2) short_backward<2>(g, dx, xf32, l.parts, st);
        else if (rb == 3) short_backward<3>(g, dx, xf32, l.parts, st);
        else short_backward<4>(g, dx, xf32, l.parts, st);
    } else {
        if (rb == 1) launch_short_logits<1, false>(g, st);
        else if (rb == 2) launch_short_logits<2, false>(g, st);
        else if (rb == 3) launch_short_logits<3, false>(g, st);
        else launch_short_logits<4, false>(g, st);
        hipLaunchKernelGGL(xent_short_join_kernel, dim3((unsigned)g.n), dim3(256), 0, st, g, loss, lse, hits, (int)short_slices(g.v));
    }
    return mgx_launch_status();
}

// Which form a call takes (both sides measured, forward + backward in us, float32):
//   few rows | a block of rows   1 x 128 x 4097 15 + 17 | 18 + 30; 4 x 128 x 65536 15 + 42 | 19 + 45; 4 x 1000 x 10001 32 + 97 | 27 + 64;
//                                16 x 128 x 4097 16 + 24 | 18 + 31; 8 x 32 x 65536 16 + 44 | 18 + 35; 8 x 300 x 1000 19 + 46 | 18 + 31;
//                                16 x 1000 x 65536 80 + 486 | 62 + 200
//   a block of rows | matrix     17 x 1000 x 65536 62 + 196 | 300 + 606; 64 x 1000 x 10001 42 + 96 | 74 + 136; 64 x 128 x 4097 16 + 37 | 23 + 38;
//                                64 x 32 x 65536 17 + 47 | 35 + 53; 128 x 1000 x 65536 171 + 492 | 300 + 611;
//                                128 x 128 x 65536 38 + 109 | 52 + 85; 128 x 1000 x 10001 74 + 174 | 73 + 135
enum { FORM_FEW, FORM_SHORT, FORM_MATRIX };
int form_of(int64_t n, int64_t e, int64_t v) {
    if (n <= 4 && e * v <= 1 << 23) return FORM_FEW;
    if (n <= FEW && e <= RC && e * v <= 1 << 20) return FORM_FEW;
    return n <= 64 || (n <= 128 && e > 128 && v >= 32768) ? FORM_SHORT : FORM_MATRIX;
}

}  // namespace

extern "C" int64_t mgx_dense_xent_workspace(int64_t n, int64_t e, int64_t v, int x_is_f32, int backward) {
    if (!sizes_ok(n, e, v)) return -1;
    if (n == 0) return 0;
    const int form = form_of(n, e, v);
    if (form == FORM_FEW) return few_bytes(n, e, v, backward != 0);
    if (form == FORM_SHORT) return short_layout(n, e, v, backward != 0).total;
    return layout(n, e, v, x_is_f32 != 0, backward != 0).total;
}

extern "C" int mgx_dense_xent_fwd(const void* x, int x_is_f32, const float* w, const float* b, const int32_t* labels,
                                  float* loss, float* lse, int32_t* hits, int64_t n, int64_t e, int64_t v,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
    if (!sizes_ok(n, e, v)) return MGX_ERR_ARG;
    if (n == 0) return MGX_OK;
    if (!x || !w || !labels || !loss || !lse || !workspace) return MGX_ERR_ARG;
    if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)workspace) & 15u) != 0) return MGX_ERR_ARG;
    const bool xf = x_is_f32 != 0;
    hipStream_t st = (hipStream_t)stream;
    const int form = form_of(n, e, v);
    if (form == FORM_FEW) {
        if (workspace_bytes < few_bytes(n, e, v, false)) return MGX_ERR_WORKSPACE;
        XentRows g = {};
        g.x = x; g.w = w; g.b = b; g.labels = labels; g.n = (int)n; g.e = (int)e; g.v = v;
        g.part = (float2*)workspace;
        g.zlab = (float*)((char*)workspace + up(up(v, 64) / 64 * n * 8, 16));
        return xf ? few_forward<true>(g, loss, lse, hits, st) : few_forward<false>(g, loss, lse, hits, st);
    }
    if (form == FORM_SHORT) {
        const ShortLayout l = short_layout(n, e, v, false);
        if (workspace_bytes < l.total) return MGX_ERR_WORKSPACE;
        XentShort g = {};
        g.x = x; g.w = w; g.b = b; g.labels = labels; g.n = (int)n; g.e = (int)e; g.v = v;
        return short_call(g, xf, l, (char*)workspace, loss, lse, hits, nullptr, false, st);
    }
    const Layout l = layout(n, e, v, xf, false);
    if (workspace_bytes < l.total) return MGX_ERR_WORKSPACE;
    char* ws = (char*)workspace;
    launch_prep(l, ws, x, xf, w, b, labels, nullptr, nullptr, n, e, v, st);
    XentGemm g = {};
    g.a[0] = (f16_t*)(ws + l.wh); g.a[1] = (f16_t*)(ws + l.wl); g.b[0] = (f16_t*)(ws + l.xh); g.b[1] = (f16_t*)(ws + l.xl);
    g.lda = g.ldb = l.ep; g.kiters = (int)(l.ep / BK);
    g.bias = (float*)(ws + l.bias); g.row = (f32x4*)(ws + l.row); g.lab = (int*)(ws + l.lab);
    g.part = (float2*)(ws + l.slices); g.zlab = (float*)(ws + l.zlab); g.np = l.np;
    if (l.narrow) {
        XentStream q = {};
        q.r[0] = g.b[0]; q.r[1] = g.b[1]; q.s[0] = g.a[0]; q.s[1] = g.a[1];
        q.row = g.row; q.bias = g.bias; q.lab = g.lab; q.tiles = (int)(l.vp / ST);
        q.part = g.part; q.zlab = g.zlab; q.ld = l.np;
        if (xf) launch_stream<2, 2, 1, MODE_FWD, 2>(l, q, l.np / l.rows_wg, l.nf, st);
        else launch_stream<1, 2, 2, MODE_FWD, 2>(l, q, l.np / l.rows_wg, l.nf, st);
    } else if (xf) {
        launch_gemm<2, 2, false, false, EPI_FWD, 4>(g, l.vp, l.np, 1, st);
    } else {
        launch_gemm<2, 1, false, false, EPI_FWD, 4>(g, l.vp, l.np, 1, st);
    }
    hipLaunchKernelGGL(xent_join_kernel, dim3((unsigned)(l.np / 32)), dim3(256), 0, st, g.part, g.zlab, b, g.lab, loss, lse, hits,
                       (long)n, (long)l.np, (long)l.nf);
    return mgx_launch_status();
}

extern "C" int mgx_dense_xent_bwd(const void* x, int x_is_f32, const float* w, const float* b, const int32_t* labels,
                                  const float* lse, const float* dloss, void* dx, float* dw, float* db, int accumulate,
                                  int64_t n, int64_t e, int64_t v, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!sizes_ok(n, e, v)) return MGX_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    if (n == 0) {
        if (!accumulate && (dw || db))
            hipLaunchKernelGGL(xent_zero_kernel, dim3(1024), dim3(256), 0, st, dw, dw ? (long)(e * v) : 0L, db, db ? (long)v : 0L);
        return mgx_launch_status();
    }
    if (!x || !w || !labels || !lse || !dloss || !workspace) return MGX_ERR_ARG;
    if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)workspace) & 15u) != 0) return MGX_ERR_ARG;
    const bool xf = x_is_f32 != 0;
    const int form = form_of(n, e, v);
    if (form == FORM_FEW) {
        if (workspace_bytes < few_bytes(n, e, v, true)) return MGX_ERR_WORKSPACE;
        XentRows g = {};
        g.x = x; g.w = w; g.b = b; g.lse = lse; g.dloss = dloss; g.labels = labels; g.n = (int)n; g.e = (int)e; g.v = v;
        g.dxp = dx ? (float*)workspace : nullptr;
        g.dw = dw; g.db = db; g.accumulate = accumulate;
        return xf ? few_backward<true>(g, dx, st) : few_backward<false>(g, dx, st);
    }
    if (form == FORM_SHORT) {
        const ShortLayout l = short_layout(n, e, v, true);
        if (workspace_bytes < l.total) return MGX_ERR_WORKSPACE;
        XentShort g = {};
        g.x = x; g.w = w; g.b = b; g.lse = lse; g.dloss = dloss; g.labels = labels; g.n = (int)n; g.e = (int)e; g.v = v;
        g.dw = dw; g.db = db; g.accumulate = accumulate;
        return short_call(g, xf, l, (char*)workspace, nullptr, nullptr, nullptr, dx, true, st);
    }
    const Layout l = layout(n, e, v, xf, true);
    if (workspace_bytes < l.total) return MGX_ERR_WORKSPACE;
    char* ws = (char*)workspace;
    launch_prep(l, ws, x, xf, w, b, labels, lse, dloss, n, e, v, st);
    f16_t *xh = (f16_t*)(ws + l.xh), *xl = (f16_t*)(ws + l.xl), *dzh = (f16_t*)(ws + l.dzh), *dzl = (f16_t*)(ws + l.dzl);
    if (l.narrow) {
        XentStream q = {};
        q.exps = (int*)(ws + l.exps); q.bias = (float*)(ws + l.bias); q.lab = (int*)(ws + l.lab);
        q.row = (f32x4*)(ws + l.row);
        f16_t *wh = (f16_t*)(ws + l.wh), *wl = (f16_t*)(ws + l.wl);
        if (dx) {
            q.r[0] = xh; q.r[1] = xl; q.s[0] = wh; q.s[1] = wl;
            q.tiles = (int)(l.vp / ST); q.out = (float*)(ws + l.dxw); q.ld = l.np;
            if (xf) launch_stream<2, 2, 1, MODE_DX, 2>(l, q, l.np / l.rows_wg, l.nx, st);
            else launch_stream<1, 2, 2, MODE_DX, 1>(l, q, l.np / l.rows_wg, l.nx, st);
        }
        const XentDxJoin j = {(float*)(ws + l.dxw), q.exps, q.row, false, dx, (int)xf, (int)l.nx, (long)(l.np * l.ep), (long)n, (int)e,
                              (int)l.ep};
        if (dw || db) {
            q.r[0] = wh; q.r[1] = wl; q.s[0] = xh; q.s[1] = xl;
            q.tiles = (int)(l.np / ST); q.out = (float*)(ws + l.slabs); q.outb = (float*)(ws + l.slabs_b); q.ld = l.vp;
            q.o = {dw, db, (long)v, (long)v, (int)e, accumulate, l.nz == 1};
            if (xf) launch_stream<2, 2, 1, MODE_DW, 2>(l, q, l.vp / 128, l.nz, st);
            else launch_stream<2, 1, 1, MODE_DW, 2>(l, q, l.vp / 128, l.nz, st);
        }
        const XentDwReduce s = {q.out, q.outb, q.exps, false, dw, db, (int)l.nz, (long)(l.ep * l.vp), (long)l.vp, (int)e, (long)v, 0L, (long)l.vp,
                                accumulate};
        const bool slabs = (dw || db) && l.nz > 1;
        if (dx || slabs) launch_joins(dx ? &j : nullptr, slabs ? &s : nullptr, st);
        return mgx_launch_status();
    }
    const XentDxJoin join = {(float*)(ws + l.dxw), (int*)(ws + l.exps), (f32x4*)(ws + l.row), true, dx, (int)xf, (int)l.nx,
                             (long)(l.np * l.ep), (long)n, (int)e, (int)l.ep};
    bool joined = false;
    for (int64_t c0 = 0; c0 < l.vp; c0 += l.vc) {
        const int64_t cnt = l.vp - c0 < l.vc ? l.vp - c0 : l.vc;
        f16_t *wh = (f16_t*)(ws + l.wh) + c0 * l.ep, *wl = (f16_t*)(ws + l.wl) + c0 * l.ep;
        XentGemm g = {};
        g.exps = (int*)(ws + l.exps);
        g.a[0] = wh; g.a[1] = wl; g.b[0] = xh; g.b[1] = xl;
        g.lda = g.ldb = l.ep; g.kiters = (int)(l.ep / BK);
        g.bias = (float*)(ws + l.bias) + c0; g.lab = (int*)(ws + l.lab); g.row = (f32x4*)(ws + l.row);
        g.dzh = dzh; g.dzl = dzl; g.ldo = l.vc; g.np = l.np; g.class0 = c0;
        if (xf) launch_gemm<2, 2, false, false, EPI_DZ, 4>(g, cnt, l.np, 1, st);
        else launch_gemm<2, 1, false, false, EPI_DZ, 4>(g, cnt, l.np, 1, st);
        if (dx) {
            XentGemm q = {};
            q.a[0] = dzh; q.a[1] = dzl; q.b[0] = wh; q.b[1] = wl;
            q.lda = l.vc; q.ldb = l.ep; q.kiters = (int)(cnt / BK);
            q.out = (float*)(ws + l.dxw); q.ldo = l.ep; q.np = l.np; q.class0 = c0;
            if (xf) launch_gemm<2, 2, false, true, EPI_DX, 4>(q, l.np, l.ep, l.nx, st);
            else launch_gemm<1, 1, false, true, EPI_DX, 4>(q, l.np, l.ep, l.nx, st);
        }
        if (dw || db) {
            // classes [a0, a1) of the piece in nz parts
            auto weights = [&](int64_t a0, int64_t a1, int64_t nz) {
                if (a0 >= a1) return;
                const int64_t vs = l.vc - l.vm, first = c0 + a0;
                XentGemm q = {};
                q.exps = g.exps;
                q.a[0] = (f16_t*)(ws + l.xsh); q.a[1] = (f16_t*)(ws + l.xsl); q.b[0] = dzh + a0; q.b[1] = dzl + a0;
                q.ones = (f16_t*)(ws + l.ones);
                q.lda = l.ep; q.ldb = l.vc; q.kiters = (int)(l.np / BK);
                q.out = (float*)(ws + l.slabs); q.outb = (float*)(ws + l.slabs_b); q.ldo = vs; q.np = l.ep * vs;
                const int64_t valid = v - first < a1 - a0 ? v - first : a1 - a0;
                q.o = {dw ? dw + first : nullptr, db ? db + first : nullptr, (long)v, (long)valid, (int)e, accumulate, nz == 1};
                if (xf) launch_gemm<2, 2, true, true, EPI_DW, 2>(q, l.ep, a1 - a0, nz, st);
                else launch_gemm<1, 2, true, true, EPI_DW, 2>(q, l.ep, a1 - a0, nz, st);
                if (nz == 1) return;
                const XentDwReduce s = {q.out, q.outb, g.exps, true, dw, db, (int)nz, (long)q.np, (long)vs, (int)e, (long)v, (long)first, (long)(a1 - a0),
                                        accumulate};
                const bool last = dx && c0 + cnt == l.vp;            // dx is complete with the last piece
                launch_joins(last ? &join : nullptr, &s, st);
                joined = joined || last;
            };
            const int64_t vm = l.vm < cnt ? l.vm : cnt;
            weights(0, vm, 1);
            weights(vm, cnt, l.nz);
        }
    }
    if (dx && !joined) launch_joins(&join, nullptr, st);
    return mgx_launch_status();
}
