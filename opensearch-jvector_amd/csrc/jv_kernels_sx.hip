// jv_kernels_sx.hip — softmax cross entropy of queries over all rows of an index, and its gradient, without keeping the logits (gfx950).
//
//   z_ij = scale q_i . v_j     lse_i = log sum_j exp z_ij     loss_i = lse_i - z_i,t(i)
//   g_ij = w_i scale (exp(z_ij - lse_i) - [j = t(i)])         dq_i = sum_j g_ij v_j         dv_j = sum_i g_ij q_i
//
// Everything is a product of rows with rows (jv_mm.h).  Forward: a workgroup walks tiles of rows for one panel of queries, and every
// lane keeps the running maximum and sum of ITS rows (one column of the accumulators is one query: no exchange until the end).
// Backward: the logits are computed again, a piece of the rows at a time, and g is written twice, by query and by row, so that both
// gradients are products of rows with rows too.  Logarithms and exponentials are base 2 inside (c = scale log2 e).
//
// bf16 operands are multiplied as they are (products exact in float32, float32 sums); g is rounded to bf16 once: 2^-9 relative for each
// term of a sum over rows or queries, the size of the gradient's own final rounding.  float32 operands and g are three bf16 planes (24 bits)
// and a product is the six plane pairs that reach 2^-24: float32's accuracy at 2.7 times the rate of its own matrix instruction.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jv_mm.h"
#include "jv_mm_out.h"

using namespace jvmm;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }

__device__ __forceinline__ uint16_t bf16_bits(float x) {
    const __bf16 b = (__bf16)x;
    return __builtin_bit_cast(uint16_t, b);
}
// the three planes of a float32
__device__ __forceinline__ void planes3(float x, uint16_t (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 3; i++) {
        const __bf16 b = (__bf16)x;
        p[i] = __builtin_bit_cast(uint16_t, b);
        x -= (float)b;
    }
}

// ---------------------------------------------------------------------------------------------
// rows -> padded bf16 planes [rows][P][kp], eight components a thread
// ---------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void jvs_pack_kernel(const T* __restrict__ x, int64_t stride, int64_t rows, int d, int kp, uint16_t* __restrict__ out) {
    constexpr int P = sizeof(T) == 4 ? 3 : 1;
    const int per = kp / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per;
        const int at = (int)(i - r * per) * 8;
        const T* row = x + r * stride;
        uint16_t p[3][8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const T v = at + e < d ? row[at + e] : (T)0.0f;
            if constexpr (P == 1) {
                p[0][e] = __builtin_bit_cast(uint16_t, v);
            } else {
                uint16_t q[3];
                planes3(v, q);
#pragma unroll
                for (int k = 0; k < 3; k++) p[k][e] = q[k];
            }
        }
#pragma unroll
        for (int k = 0; k < P; k++) {
            i32x4 o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (int)((uint32_t)p[k][2 * e] | ((uint32_t)p[k][2 * e + 1] << 16));
            *(i32x4*)(out + (r * P + k) * kp + at) = o;
        }
    }
}

// rows [rows][d] -> columns as rows [d][P][kr], zeros behind `rows`: 64 x 64 blocks through LDS
template <typename T>
__global__ __launch_bounds__(256) void jvs_pack_t_kernel(const T* __restrict__ x, int64_t stride, int rows, int d, int kr, uint16_t* __restrict__ out) {
    constexpr int P = sizeof(T) == 4 ? 3 : 1;
    __shared__ T tile[64][65];
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
    for (int i = threadIdx.x; i < 4096; i += 256) {
        const int r = i >> 6, c = i & 63;
        tile[r][c] = r0 + r < rows && c0 + c < d ? x[(int64_t)(r0 + r) * stride + c0 + c] : (T)0.0f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += 256) {
        const int c = i >> 3, r = (i & 7) * 8;
        if (c0 + c >= d) continue;
        uint16_t p[3][8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (P == 1) {
                p[0][e] = __builtin_bit_cast(uint16_t, tile[r + e][c]);
            } else {
                uint16_t q[3];
                planes3(tile[r + e][c], q);
#pragma unroll
                for (int k = 0; k < 3; k++) p[k][e] = q[k];
            }
        }
#pragma unroll
        for (int k = 0; k < P; k++) {
            i32x4 o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (int)((uint32_t)p[k][2 * e] | ((uint32_t)p[k][2 * e + 1] << 16));
            *(i32x4*)(out + ((int64_t)(c0 + c) * P + k) * kr + r0 + r) = o;
        }
    }
}

extern "C" hipError_t jvk_sx_pack(const void* x, int dtype, int64_t stride, int64_t rows, int d, int kp, uint16_t* out, hipStream_t s) {
    const int64_t want = (rows * (kp / 8) + 255) / 256;
    if (want <= 0) return hipSuccess;
    const unsigned grid = (unsigned)(want < 65536 ? want : 65536);
    if (dtype == 0) jvs_pack_kernel<float><<<grid, 256, 0, s>>>((const float*)x, stride, rows, d, kp, out);
    else jvs_pack_kernel<__bf16><<<grid, 256, 0, s>>>((const __bf16*)x, stride, rows, d, kp, out);
    return hipGetLastError();
}
extern "C" hipError_t jvk_sx_pack_t(const void* x, int dtype, int64_t stride, int rows, int d, int kr, uint16_t* out, hipStream_t s) {
    if (kr <= 0 || d <= 0) return hipSuccess;
    const dim3 grid((unsigned)(kr / 64), (unsigned)((d + 63) / 64));
    if (dtype == 0) jvs_pack_t_kernel<float><<<grid, 256, 0, s>>>((const float*)x, stride, rows, d, kr, out);
    else jvs_pack_t_kernel<__bf16><<<grid, 256, 0, s>>>((const __bf16*)x, stride, rows, d, kr, out);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------
// forward: running maximum and sum over this workgroup's tiles of rows
// ---------------------------------------------------------------------------------------------
// (m, s) and (m2, s2) joined: sums relative to the larger maximum; a side that is empty (m = -inf, s = 0) adds nothing
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2);
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    s = s * exp2_(m - ref) + s2 * exp2_(m2 - ref);
    m = top;
}

template <int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void jvs_loss_kernel(const JvSxLoss a) {
    using T = Tile<BF16, MT, NT, WM, WN>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tiles = (a.mm.M + T::TM - 1) / T::TM;
    const int split = blockIdx.x, n0 = blockIdx.y * T::TN;
    float top[NT], sum[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) top[n] = -__builtin_inff(), sum[n] = 0.0f;
    for (int t = split; t < tiles; t += a.splits) {
        f32x16 acc[MT][NT];
        T::run(a.mm, t * T::TM, n0, 0, a.mm.nk * a.mm.segs, smem, acc);
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float best = -__builtin_inff();
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float z = t * T::TM + T::row_of(m, e) < a.mm.M ? acc[m][n][e] * a.c : -__builtin_inff();
                    acc[m][n][e] = z;
                    best = fmaxf(best, z);
                }
            const float now = fmaxf(top[n], best), ref = now == -__builtin_inff() ? 0.0f : now;
            float s = sum[n] * exp2_(top[n] - ref);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int e = 0; e < 16; e++) s += exp2_(acc[m][n][e] - ref);
            top[n] = now;
            sum[n] = s;
        }
    }
    // the two halves of a wave hold different rows of the same query, and so do the WM waves of a column
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wm = w % WM;
    float* sh = (float*)smem;   // [WM][TN][2]
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; n++) {
        join(top[n], sum[n], __shfl_xor(top[n], 32, 64), __shfl_xor(sum[n], 32, 64));
        if (lane < 32) {
            sh[(wm * T::TN + T::col_of(n)) * 2] = top[n];
            sh[(wm * T::TN + T::col_of(n)) * 2 + 1] = sum[n];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < T::TN; i += T::THREADS) {
        if (n0 + i >= a.mm.N) continue;
        float m = sh[i * 2], s = sh[i * 2 + 1];
#pragma unroll
        for (int k = 1; k < WM; k++) join(m, s, sh[(k * T::TN + i) * 2], sh[(k * T::TN + i) * 2 + 1]);
        float* pm = a.part + (int64_t)split * a.mm.N + n0 + i;
        float* ps = pm + (int64_t)a.splits * a.mm.N;
        if (!a.first) join(m, s, *pm, *ps);
        *pm = m;
        *ps = s;
    }
}

extern "C" hipError_t jvk_sx_loss(const JvSxLoss* a, hipStream_t s) {
    using T = Tile<BF16, 2, 2, 2, 2>;
    const int panels = (a->mm.N + T::TN - 1) / T::TN;
    if (panels <= 0 || a->mm.M <= 0) return hipSuccess;
    if (panels > 65535 || a->splits < 1) return hipErrorInvalidValue;
    hipError_t e = hipFuncSetAttribute((const void*)jvs_loss_kernel<2, 2, 2, 2>, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
    if (e != hipSuccess) return e;
    jvs_loss_kernel<2, 2, 2, 2><<<dim3((unsigned)a->splits, (unsigned)panels), T::THREADS, T::LDS, s>>>(*a);
    return hipGetLastError();
}

// one wave a query: join the partials, take the target's logit in float32 from the rows themselves
template <typename T>
__global__ __launch_bounds__(64) void jvs_join_kernel(const float* __restrict__ part, int splits, int nq, const T* __restrict__ q, int64_t q_stride,
                                                      const T* __restrict__ v, int64_t v_stride, int d, const int32_t* __restrict__ targets,
                                                      int64_t n, float scale, float* __restrict__ loss, float* __restrict__ lse) {
    const int i = blockIdx.x, lane = threadIdx.x;
    float m = -__builtin_inff(), s = 0.0f;
    for (int k = lane; k < splits; k += 64) join(m, s, part[(int64_t)k * nq + i], part[(int64_t)(splits + k) * nq + i]);
    for (int off = 32; off >= 1; off >>= 1) join(m, s, __shfl_xor(m, off, 64), __shfl_xor(s, off, 64));
    const float total = (m + log2_(s)) * 0.69314718055994531f;
    const int t = targets ? targets[i] : -1;
    const bool known = t >= 0 && t < n;
    float dot = 0.0f;
    if (known)
        for (int k = lane; k < d; k += 64) dot = fmaf((float)q[(int64_t)i * q_stride + k], (float)v[(int64_t)t * v_stride + k], dot);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) dot += __shfl_xor(dot, off, 64);
    if (lane == 0) {
        lse[i] = total;
        loss[i] = known ? total - scale * dot : 0.0f;
    }
}

extern "C" hipError_t jvk_sx_join(const float* part, int splits, int nq, const void* q, int64_t q_stride, const void* v, int64_t v_stride, int dtype,
                                  int d, const int32_t* targets, int64_t n, float scale, float* loss, float* lse, hipStream_t s) {
    if (nq <= 0) return hipSuccess;
    if (dtype == 0)
        jvs_join_kernel<float><<<nq, 64, 0, s>>>(part, splits, nq, (const float*)q, q_stride, (const float*)v, v_stride, d, targets, n, scale, loss, lse);
    else
        jvs_join_kernel<__bf16><<<nq, 64, 0, s>>>(part, splits, nq, (const __bf16*)q, q_stride, (const __bf16*)v, v_stride, d, targets, n, scale, loss, lse);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------
// backward: the logits again, as weights g
// ---------------------------------------------------------------------------------------------
template <int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void jvs_weights_kernel(const JvSxWeights a) {
    using T = Tile<BF16, MT, NT, WM, WN>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int m0 = blockIdx.x * T::TM, n0 = blockIdx.y * T::TN;
    f32x16 acc[MT][NT];
    T::run(a.mm, m0, n0, 0, a.mm.nk * a.mm.segs, smem, acc);
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int col = n0 + T::col_of(n);
        const bool live = col < a.mm.N;
        const int t = live ? a.targets[col] : -1;
        const bool known = t >= 0 && t < a.n;
        const float w = known ? (a.w ? a.w[col] : 1.0f) * a.scale : 0.0f;
        const float lse2 = known ? a.lse[col] * 1.44269504088896341f : 0.0f;
        const int at = known && t >= a.row0 && t - a.row0 < a.mm.M ? (int)(t - a.row0) : -1;
#pragma unroll
        for (int m = 0; m < MT; m++) {
#pragma unroll
            for (int e4 = 0; e4 < 4; e4++) {
                uint16_t p[4][3];
                const int row = m0 + T::row_of(m, e4 * 4);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float g = exp2_(fmaf(acc[m][n][e4 * 4 + e], a.c, -lse2)) - (row + e == at ? 1.0f : 0.0f);
                    g = known && row + e < a.mm.M ? g * w : 0.0f;
                    planes3(g, p[e]);
                }
#pragma unroll
                for (int k = 0; k < 3; k++) {
                    if (k >= a.planes) break;
                    if (a.g && live && row < a.kv)   // (kv is a multiple of 64: four rows are in or out together)
                        *(uint2*)(a.g + ((int64_t)col * a.planes + k) * a.kv + row) =
                            make_uint2((uint32_t)p[0][k] | ((uint32_t)p[1][k] << 16), (uint32_t)p[2][k] | ((uint32_t)p[3][k] << 16));
                    if (a.gt && col < a.kq) {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (row + e < a.mm.M) a.gt[((int64_t)(row + e) * a.planes + k) * a.kq + col] = p[e][k];
                    }
                }
            }
        }
    }
}

extern "C" hipError_t jvk_sx_weights(const JvSxWeights* a, hipStream_t s) {
    using T = Tile<BF16, 2, 2, 2, 2>;
    if (a->mm.M <= 0 || a->mm.N <= 0) return hipSuccess;
    const int panels = (a->mm.N + T::TN - 1) / T::TN;
    if (panels > 65535) return hipErrorInvalidValue;
    hipError_t e = hipFuncSetAttribute((const void*)jvs_weights_kernel<2, 2, 2, 2>, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
    if (e != hipSuccess) return e;
    jvs_weights_kernel<2, 2, 2, 2><<<dim3((unsigned)((a->mm.M + T::TM - 1) / T::TM), (unsigned)panels), T::THREADS, T::LDS, s>>>(*a);
    return hipGetLastError();
}

extern "C" hipError_t jvk_sx_mm(const JvMmOut* a, hipStream_t s) { return mm_out<BF16, 2, 2, 2, 2>(*a, s); }

// partial sums -> the gradient's rows
template <typename T>
__global__ __launch_bounds__(256) void jvs_finish_kernel(const float* __restrict__ slab, int splits, int64_t rows, int d, T* __restrict__ out, int64_t ldo) {
    const int64_t all = rows * d;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        float v = 0.0f;
        for (int k = 0; k < splits; k++) v += slab[k * all + i];
        const int64_t r = i / d;
        out[r * ldo + (i - r * d)] = (T)v;
    }
}
template <typename T>
__global__ __launch_bounds__(256) void jvs_fill_kernel(T* __restrict__ out, int64_t stride, int64_t rows, int d, float value) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * d; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / d;
        out[r * stride + (i - r * d)] = (T)value;
    }
}
static unsigned grid_for(int64_t items) {
    const int64_t want = (items + 255) / 256;
    return (unsigned)(want < 16384 ? want : 16384);
}
extern "C" hipError_t jvk_sx_finish(const float* slab, int splits, int64_t rows, int d, void* out, int dtype, int64_t ldo, hipStream_t s) {
    if (rows <= 0 || d <= 0) return hipSuccess;
    if (dtype == 0) jvs_finish_kernel<float><<<grid_for(rows * d), 256, 0, s>>>(slab, splits, rows, d, (float*)out, ldo);
    else jvs_finish_kernel<__bf16><<<grid_for(rows * d), 256, 0, s>>>(slab, splits, rows, d, (__bf16*)out, ldo);
    return hipGetLastError();
}
extern "C" hipError_t jvk_sx_fill(void* out, int dtype, int64_t stride, int64_t rows, int d, float value, hipStream_t s) {
    if (rows <= 0 || d <= 0) return hipSuccess;
    if (dtype == 0) jvs_fill_kernel<float><<<grid_for(rows * d), 256, 0, s>>>((float*)out, stride, rows, d, value);
    else jvs_fill_kernel<__bf16><<<grid_for(rows * d), 256, 0, s>>>((__bf16*)out, stride, rows, d, value);
    return hipGetLastError();
}
