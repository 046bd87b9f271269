// jv_tile3.h — float32 products of middling size: A as three bf16 planes, B as it lies.
//
// As in jv_tile32.h a float32 value is three bf16 parts and a product the six pairs that reach 2^-24.  There both operands are split by every
// wave that needs them, which costs as much as the multiplications.  Here the operand that many tiles share (the queries, or g, which is
// written that way) comes as planes [rows][3][k], and the other one is split by the one wave that holds it: a workgroup's four waves lie
// side by side along N, MT accumulators of 32 x 32 each.  k goes by in steps of 32, two in LDS (80 KB with MT = 4: two workgroups a CU).
//   A, k along its rows:  64 B a row and plane, piece p (16 B) of row r at p ^ ((r >> 2) & 3);
//   A, k across (TA):     32 rows of TM columns a plane, read through the transposing read, piece p of row k at p ^ ((k & 3) << 2);
//   B, k along its rows:  128 B a row, piece p of row r at p ^ ((r >> 1) & 7);      all: 16 consecutive rows cover the 64 banks once
//   B, k across (TB):     32 rows of 128 columns, rows 8 .. 15 and 24 .. 31 with their halves of 256 B swapped.
// Bound by the matrix unit and the splitting beside it: loss 777 x 30 011 x 381 160 us, 670 TFLOP/s of bf16 products (the unit is busy half of the cycles); with
// few queries by the rows' bytes (loss 11 x 257 776 x 1272: 268 us, 4.9 TB/s).  Three buffers, or three workgroups a CU, changed nothing.
#pragma once
#include "jv_tile32.h"

namespace jvmm {

template <int MT_, bool TA, bool TB>
struct Tile3 {
    using acc_t = f32x16;
    static constexpr bool RAW = false;
    static constexpr int RESIDENT = 2;   // workgroups a CU
    static constexpr int E = 16, WIDE = 32;
    static constexpr int MT = MT_, NT = 1, WAVES = 4, THREADS = 256, TM = 32 * MT, TN = 128;
    static constexpr int KA = 6 * MT, PA = (KA + 3) / 4, PB = 4, PER = PA + PB;   // KB of A in a step; copies of one wave (the last of A twice, if need be)
    static constexpr int BUF = (KA + 16) * 1024, LDS = 2 * BUF;
    static_assert(!TA || MT == 4, "a plane's rows of 256 B");
    static __host__ __device__ __forceinline__ int steps(const JvMm& a) { return (a.k + 31) / 32; }
    using Split = Tile32<1, 1, 1, 4, 2, false, false>;

    static __device__ __forceinline__ bf16x8 part_a(const unsigned char* base, int t, int plane, int kk) {
        const int lane = threadIdx.x & 63, h = lane >> 5, r31 = lane & 31;
        if constexpr (!TA) {
            const int r = t * 32 + r31;
            return *(const bf16x8*)(base + (plane * TM + r) * 64 + (((2 * kk + h) ^ ((r >> 2) & 3)) << 4));
        } else {
            const int c = t * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4, tk = (lane & 15) >> 2;
            const unsigned char* p = base + (plane * 32 + 16 * kk + 8 * h + tk) * 256 + (((c >> 3) ^ (tk << 2)) << 4) + (c & 4) * 2;
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(read_across(p), read_across(p + 4 * 256), 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
    // eight k's of this wave's row or column of B, in three parts
    template <bool LAST>
    static __device__ __forceinline__ void part_b(const unsigned char* base, int r, int kk, int valid, int k, bf16x8 (&p)[3]) {
        const int h = (threadIdx.x >> 5) & 1;
        float x[8];
        if constexpr (!TB) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int piece = 4 * kk + 2 * h + half;
                f32x4 v = *(const f32x4*)(base + r * 128 + ((piece ^ ((r >> 1) & 7)) << 4));
                if constexpr (LAST) v = Split::tail(v, piece, valid, k);
#pragma unroll
                for (int e = 0; e < 4; e++) x[4 * half + e] = v[e];
            }
        } else {
            const int c = r ^ (h << 5);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = *(const float*)(base + (16 * kk + 8 * h + e) * 512 + c * 4);
        }
        Split::split(x, p);
    }
    template <bool LAST>
    static __device__ __forceinline__ void multiply(const JvMm& a, const unsigned char* base, int rb, int valid, f32x16 (&acc)[MT][1]) {
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            bf16x8 va[MT][3], vb[3];
            part_b<LAST>(base + KA * 1024, rb, kk, valid, a.k, vb);
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int p = 0; p < 3; p++) va[t][p] = part_a(base, t, p, kk);
#pragma unroll
            for (int g = 0; g < 6; g++) {
                const int pa = part_of_a(g), pb = part_of_b(g);
#pragma unroll
                for (int m = 0; m < MT; m++) acc[m][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb[pb], va[m][pa], acc[m][0], 0, 0, 0);
            }
        }
    }

    // C tile at (m0, n0), steps [k0, k1) of ceil(k / 32); A's planes hold zeros behind component k, B is masked there
    static __device__ __forceinline__ void run(const JvMm& a, int m0, int n0, int k0, int k1, unsigned char* smem, f32x16 (&acc)[MT][1]) {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r31 = lane & 31;
        const char *pa[PA], *pb[PB];
#pragma unroll
        for (int i = 0; i < PA; i++) {
            const int c = min(i * 4 + w, KA - 1);   // KB of A: 16 rows of a plane (k along), or four of its 32 rows (k across)
            if constexpr (!TA) {
                const int plane = c / (2 * MT), r = (c - plane * 2 * MT) * 16 + (lane >> 2);
                pa[i] = a.a + plane * a.plane_a + (int64_t)min(m0 + r, a.M - 1) * a.lda + ((lane & 3) ^ ((r >> 2) & 3)) * 16;
            } else {
                const int plane = c >> 3, k = (c & 7) * 4 + (lane >> 4);
                pa[i] = a.a + plane * a.plane_a + (int64_t)min(m0 + 8 * ((lane & 15) ^ ((k & 3) << 2)), a.ca - 8) * 2;
            }
        }
#pragma unroll
        for (int i = 0; i < PB; i++) {
            const int c = i * 4 + w;
            if constexpr (!TB) {
                pb[i] = a.b + (int64_t)min(n0 + 8 * c + (lane >> 3), a.N - 1) * a.ldb;
            } else {
                const int k = 2 * c + (lane >> 5);
                pb[i] = a.b + (int64_t)min(n0 + (((lane & 31) << 2) ^ (((k >> 3) & 1) << 5)), max(a.cb, 4) - 4) * 4;
            }
        }
        const int rb = TB ? Tile32<2, 2, 2, 2, 2, false, true>::template Side<true, 16>::place(w * 32 + r31, n0, a.cb) : w * 32 + r31;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[m][0][e] = 0.0f;
        auto stage = [&](int s) {
            unsigned char* dst = smem + ((s - k0) & 1) * BUF;
#pragma unroll
            for (int i = 0; i < PA; i++) {
                const int c = min(i * 4 + w, KA - 1);
                const int64_t off = TA ? (int64_t)min(s * 32 + (c & 7) * 4 + (lane >> 4), a.ka - 1) * a.lda : (int64_t)s * 64;
                glds16(pa[i] + off, dst + c * 1024);
            }
#pragma unroll
            for (int i = 0; i < PB; i++) {
                const int c = i * 4 + w;
                int64_t off;
                if constexpr (!TB) off = (int64_t)min(s * 32 + (((lane & 7) ^ ((4 * c + (lane >> 4)) & 7)) << 2), max(a.k, 4) - 4) * 4;
                else off = (int64_t)min(s * 32 + 2 * c + (lane >> 5), a.kb - 1) * a.ldb;
                glds16(pb[i] + off, dst + (KA + c) * 1024);
            }
        };
        stage(k0);
        for (int s = k0; s < k1; s++) {
            if (s + 1 < k1) stage(s + 1);
            wait_step<2, PER>(k1 - 1 - s);
            const unsigned char* base = smem + ((s - k0) & 1) * BUF;
            if (TB || (s + 1) * 32 <= a.k) multiply<false>(a, base, rb, 32, acc);
            else multiply<true>(a, base, rb, a.k - s * 32, acc);
            release_step<false>();
        }
    }
    // acc[m][0][e] is C[row(m)][col(0, e)] of the tile, four consecutive e are four consecutive columns
    static __device__ __forceinline__ int row(int m) { return m * 32 + (threadIdx.x & 31); }
    static __device__ __forceinline__ int col(int, int e) { return (threadIdx.x >> 6) * 32 + (e & 3) + 8 * (e >> 2) + 4 * ((threadIdx.x >> 5) & 1); }
};

}  // namespace jvmm
