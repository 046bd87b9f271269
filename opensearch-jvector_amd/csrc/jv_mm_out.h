// jv_mm_out.h — the product of jv_mm.h written as it is: rows of float32 or bf16, or float32 partial sums of a split k range.
#pragma once
#include "jv_mm.h"

namespace jvmm {

// The workgroups of one XCD (blockIdx % 8 of the grid) take a contiguous run of tiles, A's tiles innermost: what they share of B meets
// in one L2 (bijective for any grid size).
__device__ __forceinline__ int xcd_order(int i, int n) {
    const int xcd = i & 7, slot = i >> 3, q = n >> 3, r = n & 7;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + slot;
}

template <int TY, int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void jvm_out_kernel(const JvMmOut a) {
    using T = Tile<TY, MT, NT, WM, WN>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tm = (a.mm.M + T::TM - 1) / T::TM;
    const int L = xcd_order(blockIdx.x, gridDim.x);
    const int m0 = (L % tm) * T::TM, n0 = (L / tm) * T::TN;
    const int steps = a.mm.nk * a.mm.segs;
    const int k0 = (int)((int64_t)steps * blockIdx.y / a.splits), k1 = (int)((int64_t)steps * (blockIdx.y + 1) / a.splits);
    f32x16 acc[MT][NT];
    T::run(a.mm, m0, n0, k0, k1, smem, acc);
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int col = n0 + T::col_of(n);
        if (col >= a.mm.N) continue;
#pragma unroll
        for (int m = 0; m < MT; m++) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int row = m0 + T::row_of(m, e);
                if (row >= a.mm.M) continue;
                const float v = acc[m][n][e];
                if (a.slab) {
                    float* p = a.slab + ((int64_t)blockIdx.y * a.mm.M + row) * a.mm.N + col;
                    *p = a.add ? *p + v : v;
                } else if (a.dtype == 0) {
                    ((float*)a.out)[(int64_t)row * a.ldo + col] = v;
                } else {
                    ((__bf16*)a.out)[(int64_t)row * a.ldo + col] = (__bf16)v;
                }
            }
        }
    }
}

template <int TY, int MT, int NT, int WM, int WN>
static hipError_t mm_out(const JvMmOut& a, hipStream_t s) {
    using T = Tile<TY, MT, NT, WM, WN>;
    if (a.mm.M <= 0 || a.mm.N <= 0) return hipSuccess;
    const int64_t tiles = (int64_t)((a.mm.M + T::TM - 1) / T::TM) * ((a.mm.N + T::TN - 1) / T::TN);
    if (tiles > 0x7fffffffll || a.splits < 1 || a.splits > 65535 || a.splits > a.mm.nk * a.mm.segs) return hipErrorInvalidValue;
    hipError_t e = hipFuncSetAttribute((const void*)jvm_out_kernel<TY, MT, NT, WM, WN>, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
    if (e != hipSuccess) return e;
    jvm_out_kernel<TY, MT, NT, WM, WN><<<dim3((unsigned)tiles, (unsigned)a.splits), T::THREADS, T::LDS, s>>>(a);
    return hipGetLastError();
}

}  // namespace jvmm
