// jv_mm.h — the matrix-core product of rows with rows that the training and 8-bit scoring kernels share (see JvMm).
//
// A workgroup owns a tile of C and walks k in steps of 128 bytes a row, in one of three kinds of arithmetic:
//   BF16  64 bf16 (v_mfma_f32_32x32x16_bf16: exact products, float32 sums);
//   F8    128 e4m3 as they are (v_mfma_scale_f32_32x32x64_f8f6f4, whose operands take the block's power-of-two scale as an exponent byte:
//         the scale costs no vector instruction).  This unit adds a group's products with about 12 bits below the largest of them
//         (measured: off by up to 2^-11.7 of the largest product, 1.4e-5 of the result's norm), so it serves results of 8 bits;
//   F8W   128 e4m3 widened to bf16 with their scale on the way into the bf16 unit (exact: 4 significant bits): float32 sums (5e-8 of the
//         result's norm) at half the rate and one conversion for every two components.
// Both operands are staged with 16-B copies straight into LDS; a copy's 64 lanes fill an 8-row group of 1 024 B in
// order, so the swizzle (16-B piece p of row r at p ^ (r & 7)) is on the source address.  Groups are 1 152 B apart: a 16-B fragment
// read serves 16 consecutive rows at a time, the pad puts the two groups of such a pair on opposite halves of the 256-B bank row.
// Bound by the rows' bytes with few queries (loss 8 x 87 332 x 384, bf16: 14 us, 4.8 TB/s), by the way through a tile's steps where there are few
// tiles (loss 2048 x 2048 x 768: 18 us, 360 TFLOP/s).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jv_ops.h"

namespace jvmm {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;

enum { BF16 = 0, F8 = 1, F8W = 2 };
constexpr int GROUP = 1152;

__device__ __forceinline__ void glds16(const char* g, unsigned char* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// eight e4m3 codes times 2^(byte - 127), as bf16
__device__ __forceinline__ bf16x8 widen(int lo, int hi, int byte) {
    const float s = __int_as_float(byte << 23);
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    const bf16x4 x = __builtin_shufflevector(a, b, 0, 1, 2, 3), y = __builtin_shufflevector(c, d, 0, 1, 2, 3);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

typedef __attribute__((ext_vector_type(4))) short s16x4;
__device__ __forceinline__ s16x4 read_across(const unsigned char* p) {   // 16 lanes give four rows of 16 columns, and take a column's four rows
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

// This wave's copies of a step have landed and everybody's have (SOLO: a wave with LDS of its own), `left` steps (PER copies each, NS - 1 at most)
// being under way behind it.
template <int NS, int PER, bool SOLO = false>
__device__ __forceinline__ void wait_step(int left) {
    static_assert(NS >= 2 && NS <= 4);
    constexpr int most = 63;   // (what the counter holds)
    if (left >= NS - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * PER < most ? (NS - 1) * PER : most) : "memory");
    else if (NS > 3 && left == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PER < most ? 2 * PER : most) : "memory");
    else if (NS > 2 && left == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER < most ? PER : most) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (!SOLO) asm volatile("s_barrier" ::: "memory");
}
// Every fragment read of a buffer has returned before any wave stages into it again.
template <bool SOLO>
__device__ __forceinline__ void release_step() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (!SOLO) asm volatile("s_barrier" ::: "memory");
}

// The product for small shapes: MT x NT accumulators of 32 x 32 for each of WM x WN waves, NS steps of k in LDS: two and
// several workgroups a CU, or four where there are no more workgroups than CUs and the way to memory is what counts.
// TA / TB: an operand with k across its rows (bf16): 64 rows of TM / TN columns a step.  Four rows of 64 B are read at a time: piece p of row k
// lies at p ^ (swirl << 2) so that they are the four quarters of a 256-B bank row.
template <int TY, int MT_, int NT_, int WM, int WN, int NS, bool TA = false, bool TB = false>
struct Tile {
    using acc_t = f32x16;
    static constexpr bool RAW = false;
    static constexpr int MT = MT_, NT = NT_, RESIDENT = 1, E = 16, WIDE = 32 * NT;   // values of an accumulator; columns of a wave
    static constexpr int TM = 32 * MT * WM, TN = 32 * NT * WN, WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int GA = TM / 8, GB = TN / 8;                               // 8-row groups
    static constexpr int CA = GA / WAVES, CB = GB / WAVES, PER = CA + CB;        // copies of one wave a step
    static constexpr int BUF = (GA + GB) * GROUP, LDS = NS * BUF;
    static_assert(GA % WAVES == 0 && GB % WAVES == 0, "every wave copies the same number of groups of each operand");
    static_assert(TY == BF16 || (!TA && !TB), "8-bit operands have k along their rows");
    static __host__ __device__ __forceinline__ int steps(const JvMm& a) { return a.kph >> 1; }

    template <int PIECES>   // 16-B pieces of a row
    static __device__ __forceinline__ int swirl(int k) {
        return PIECES >= 16 ? k & 3 : PIECES == 8 ? (k >> 1) & 1 : 0;
    }
    // 32 columns from `first` on, rows 16 kk + 8 h + (0 .. 7)
    template <int PIECES>
    static __device__ __forceinline__ bf16x8 across(const unsigned char* base, int first, int kk) {
        const int lane = threadIdx.x & 63, c = first + ((lane >> 4) & 1) * 16 + (lane & 3) * 4, k = 16 * kk + 8 * (lane >> 5) + ((lane & 15) >> 2);
        auto at = [&](int row) { return base + (row * PIECES + ((c >> 3) ^ (swirl<PIECES>(row) << 2))) * 16 + (c & 4) * 2; };
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(read_across(at(k)), read_across(at(k + 4)), 0, 1, 2, 3, 4, 5, 6, 7));
    }

    // C tile at (m0, n0), steps [k0, k1).  Rows behind the operands' last are read as their last.
    static __device__ __forceinline__ void run(const JvMm& a, int m0, int n0, int k0, int k1, unsigned char* smem, f32x16 (&acc)[MT][NT]) {
        const int nk = a.kph >> 1;   // scales of a row
        const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
        const int lr = lane >> 3, lp = (lane & 7) ^ lr;
        const char* src[PER];   // k along rows: the row's piece; k across: the column's piece of row 0
        int krow[PER];          // k across: the row inside a step
        bool ends[CB];          // k across: this piece is the last of B's row
#pragma unroll
        for (int i = 0; i < CA; i++) {
            krow[i] = (i * WAVES + w) * (64 / GA) + lane / GA;   // (a row of TM columns is GA pieces)
            if constexpr (!TA) src[i] = a.a + (int64_t)min(m0 + 8 * (i * WAVES + w) + lr, a.M - 1) * a.lda + lp * 16;
            else src[i] = a.a + (int64_t)min(m0 + 8 * ((lane % GA) ^ (swirl<GA>(krow[i]) << 2)), a.ca - 8) * 2;
        }
#pragma unroll
        for (int i = 0; i < CB; i++) {
            krow[CA + i] = (i * WAVES + w) * (64 / GB) + lane / GB;
            if constexpr (!TB) src[CA + i] = a.b + (int64_t)min(n0 + 8 * (i * WAVES + w) + lr, a.N - 1) * a.ldb + lp * 16;
            else {
                const int col = min(n0 + 8 * ((lane % GB) ^ (swirl<GB>(krow[CA + i]) << 2)), a.cb - 8);
                src[CA + i] = a.b + (int64_t)col * 2, ends[i] = a.tail_b && col == a.cb - 8;
            }
        }
        const int wm = w % WM, wn = w / WM, h = lane >> 5, r31 = lane & 31;
        int aoff[MT], boff[NT], ax, bx;
#pragma unroll
        for (int t = 0; t < MT; t++) {
            const int r = (wm * MT + t) * 32 + r31;
            aoff[t] = (r >> 3) * GROUP + (r & 7) * 128;
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int r = (wn * NT + t) * 32 + r31;
            boff[t] = (GA + (r >> 3)) * GROUP + (r & 7) * 128;
        }
        ax = bx = r31 & 7;
        const uint8_t *pa[MT], *pb[NT];
        if constexpr (TY != BF16) {
#pragma unroll
            for (int t = 0; t < MT; t++) pa[t] = a.sa + (int64_t)min(m0 + (wm * MT + t) * 32 + r31, a.M - 1) * nk;
#pragma unroll
            for (int t = 0; t < NT; t++) pb[t] = a.sb + (int64_t)min(n0 + (wn * NT + t) * 32 + r31, a.N - 1) * nk;
        }
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[m][n][e] = 0.0f;

        int kin = k0;   // the next step to be staged
        auto stage = [&](int buf) {
            const int64_t off = (int64_t)kin * 128;
            unsigned char* dst = smem + buf * BUF;
#pragma unroll
            for (int i = 0; i < CA; i++)
                glds16(src[i] + (TA ? (int64_t)min(kin * 64 + krow[i], a.ka - 1) * a.lda : off), dst + (i * WAVES + w) * (TA ? 1024 : GROUP));
#pragma unroll
            for (int i = 0; i < CB; i++) {
                const int k = kin * 64 + krow[CA + i];
                const char* p = src[CA + i] + (TB ? (int64_t)min(k, a.kb - 1) * a.ldb : min(off, (int64_t)(a.end_b - 16 - lp * 16)));
                if (TB && ends[i] && k >= a.kb - 1) p = a.tail_b;
                glds16(p, dst + GA * GROUP + (i * WAVES + w) * (TB ? 1024 : GROUP));
            }
            kin++;
        };
#pragma unroll
        for (int i = 0; i < NS - 1; i++)
            if (k0 + i < k1) stage(i);
        int buf = 0;
        for (int s = k0; s < k1; s++) {
            int fa[MT], fb[NT];
            if constexpr (TY != BF16) {
#pragma unroll
                for (int t = 0; t < MT; t++) fa[t] = pa[t][s];
#pragma unroll
                for (int t = 0; t < NT; t++) fb[t] = pb[t][s];
            }
            if (s + NS - 1 < k1) stage(buf == 0 ? NS - 1 : buf - 1);
            wait_step<NS, PER>(k1 - 1 - s);
            const unsigned char* base = smem + buf * BUF;
            if constexpr (TY == BF16) {
#pragma unroll
                for (int kk = 0; kk < 4; kk++) {
                    bf16x8 va[MT], vb[NT];
#pragma unroll
                    for (int t = 0; t < MT; t++) {
                        if constexpr (TA) va[t] = across<GA>(base, (wm * MT + t) * 32, kk);
                        else va[t] = *(const bf16x8*)(base + aoff[t] + (((2 * kk + h) ^ ax) << 4));
                    }
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        if constexpr (TB) vb[t] = across<GB>(base + GA * GROUP, (wn * NT + t) * 32, kk);
                        else vb[t] = *(const bf16x8*)(base + boff[t] + (((2 * kk + h) ^ bx) << 4));
                    }
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int n = 0; n < NT; n++) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb[n], va[m], acc[m][n], 0, 0, 0);
                }
            } else if constexpr (TY == F8W) {
                // (16 components a lane and step: which of the block's 128 does not matter as long as both operands agree)
#pragma unroll
                for (int kk = 0; kk < 4; kk++) {
                    i32x4 ra[MT], rb[NT];
#pragma unroll
                    for (int t = 0; t < MT; t++) ra[t] = *(const i32x4*)(base + aoff[t] + (((2 * kk + h) ^ ax) << 4));
#pragma unroll
                    for (int t = 0; t < NT; t++) rb[t] = *(const i32x4*)(base + boff[t] + (((2 * kk + h) ^ bx) << 4));
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        bf16x8 va[MT], vb[NT];
#pragma unroll
                        for (int t = 0; t < MT; t++) va[t] = widen(ra[t][2 * half], ra[t][2 * half + 1], fa[t]);
#pragma unroll
                        for (int t = 0; t < NT; t++) vb[t] = widen(rb[t][2 * half], rb[t][2 * half + 1], fb[t]);
#pragma unroll
                        for (int m = 0; m < MT; m++)
#pragma unroll
                            for (int n = 0; n < NT; n++) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb[n], va[m], acc[m][n], 0, 0, 0);
                    }
                }
            } else {
                // (which 32 of the block's 128 components a lane holds does not matter as long as both operands agree: one scale for all)
#pragma unroll
                for (int kk = 0; kk < 2; kk++) {
                    i32x8 va[MT], vb[NT];
                    auto frag = [&](int off, int x) -> i32x8 {
                        const i32x4 lo = *(const i32x4*)(base + off + (((4 * kk + 2 * h) ^ x) << 4));
                        const i32x4 hi = *(const i32x4*)(base + off + (((4 * kk + 2 * h + 1) ^ x) << 4));
                        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    };
#pragma unroll
                    for (int t = 0; t < MT; t++) va[t] = frag(aoff[t], ax);
#pragma unroll
                    for (int t = 0; t < NT; t++) vb[t] = frag(boff[t], bx);
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int n = 0; n < NT; n++)
                            acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(vb[n], va[m], acc[m][n], 0, 0, 0, fb[n], 0, fa[m]);
                }
            }
            release_step<false>();
            buf = buf + 1 == NS ? 0 : buf + 1;
        }
    }
    // acc[m][n][e] is C[row(m)][col(n, e)] of the tile, four consecutive e are four consecutive columns
    static __device__ __forceinline__ int row(int m) { return (((threadIdx.x >> 6) % WM) * MT + m) * 32 + (threadIdx.x & 31); }
    static __device__ __forceinline__ int col(int n, int e) {
        return (((threadIdx.x >> 6) / WM) * NT + n) * 32 + (e & 3) + 8 * (e >> 2) + 4 * ((threadIdx.x >> 5) & 1);
    }
};

}  // namespace jvmm
