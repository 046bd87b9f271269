// jv_tile32.h — the product of jv_mm.h for small shapes whose operands are float32 as they lie in memory.
//
// A float32 product on the bf16 matrix unit: each operand is split into three bf16 parts (x = h + m + l, 24 bits) on the way from LDS into the
// fragments, and the six pairs of parts that reach 2^-24 are multiplied, the smallest first.  Nothing is laid out beforehand: a value is read
// from memory once for each tile that needs it, as 4 bytes, where planes in memory would be written as 6 and read as 12.  k goes by in steps
// of 32; LDS holds NS of them (Tile).  An operand with k along its rows (d components, any number: what lies behind is masked in the last step) is
// staged in 8-row groups of 128 B a row as in Tile; one with k across its rows as 32 rows of TM / TN columns, where the rows 8 .. 15 and
// 24 .. 31 have their 128-B halves of 256 B swapped, so that the two halves of a wave, eight rows apart, read different banks.
// Copies are 16 B a lane, or 4 B (NA / NB) where a row is not 16-B aligned or ends inside 16 B.
#pragma once
#include "jv_mm.h"

namespace jvmm {

template <int MT_, int NT_, int WM, int WN, int NS, bool TA, bool TB, bool NA, bool NB>
struct Tile32 {
    static constexpr int MT = MT_, NT = NT_;
    static constexpr int TM = 32 * MT * WM, TN = 32 * NT * WN, WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int GA = TM / 8, GB = TN / 8;                       // KB of a step
    static constexpr int CA = GA / WAVES * (NA ? 4 : 1), CB = GB / WAVES * (NB ? 4 : 1), PER = CA + CB;   // copies of one wave a step
    static constexpr int BUF = (GA + GB) * GROUP, LDS = NS * BUF, AHEAD = (NS - 1) * PER < 63 ? (NS - 1) * PER : 63;
    static_assert(GA % WAVES == 0 && GB % WAVES == 0, "every wave copies the same number of groups of each operand");
    static_assert((!TA || GA >= 8) && (!TB || GB >= 8), "the swapped halves are 32 columns each");
    static __device__ __forceinline__ int steps(const JvMm& a) { return (a.k + 31) / 32; }

    static __device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&p)[3]) {
        float r[8];
#pragma unroll
        for (int e = 0; e < 8; e++) r[e] = x[e];
#pragma unroll
        for (int k = 0; k < 3; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                p[k][e] = (__bf16)r[e];
                if (k < 2) r[e] -= (float)p[k][e];
            }
    }

    // One operand of `rows` rows (k along) or columns (k across), ROWS = TM / TN of them from `first` on.
    template <bool ACROSS, bool NARROW, int GROUPS>
    struct Side {
        static constexpr int COPIES = GROUPS / WAVES * (NARROW ? 4 : 1);
        static constexpr int STRIDE = ACROSS ? 1024 : GROUP;   // LDS bytes of a KB of the operand
        const char* src[COPIES];

        // copy i of this wave is number c = i * WAVES + w of its KB (wide) or 256 B (narrow)
        __device__ __forceinline__ void init(const char* base, int64_t ld, int first, int rows, int cols) {
            const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
            for (int i = 0; i < COPIES; i++) {
                const int c = i * WAVES + w;
                if constexpr (!ACROSS) {
                    const int row = NARROW ? 2 * c + (lane >> 5) : 8 * c + (lane >> 3);
                    src[i] = base + (int64_t)min(first + row, rows - 1) * ld;
                } else {
                    const int byte = NARROW ? c * 256 + lane * 4 : c * 1024 + lane * 16, k = byte / (GROUPS * 32);
                    const int col = ((byte % (GROUPS * 32)) >> 2) ^ (((k >> 3) & 1) << 5);
                    src[i] = base + (int64_t)min(first + col, cols - (NARROW ? 1 : 4)) * 4;
                }
            }
        }
        __device__ __forceinline__ void copy(int64_t ld, int step, int k, unsigned char* dst) {
            const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
            for (int i = 0; i < COPIES; i++) {
                const int c = i * WAVES + w;
                const char* p = src[i];
                if constexpr (!ACROSS) {
                    // piece (16 B) or component inside the 128 B of a row; what lies behind the last component reads as the first (and is masked)
                    const int row = NARROW ? 2 * c + (lane >> 5) : 8 * c + (lane >> 3);
                    const int at = NARROW ? ((((lane & 31) >> 2) ^ (row & 7)) << 2) + (lane & 3) : ((lane & 7) ^ (row & 7)) << 2;
                    const int col = step * 32 + at;
                    p += (int64_t)(col < k ? col : 0) * 4;
                } else {
                    const int byte = NARROW ? c * 256 + lane * 4 : c * 1024 + lane * 16, row = byte / (GROUPS * 32);
                    p += (int64_t)min(step * 32 + row, k - 1) * ld;
                }
                if constexpr (NARROW) {
                    unsigned char* to = dst + (ACROSS ? c * 256 : (c >> 2) * GROUP + (c & 3) * 256);
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)to, 4, 0, 0);
                } else {
                    glds16(p, dst + c * STRIDE);
                }
            }
        }
        // eight k's (16 kk + 8 h ..) of row or column r; `valid`: components of this step (k along rows)
        __device__ __forceinline__ void read(const unsigned char* base, int r, int kk, int valid, bf16x8 (&p)[3]) const {
            const int h = (threadIdx.x >> 5) & 1;
            float x[8];
            if constexpr (!ACROSS) {
                const unsigned char* row = base + (r >> 3) * GROUP + (r & 7) * 128;
                *(f32x4*)x = *(const f32x4*)(row + (((4 * kk + 2 * h) ^ (r & 7)) << 4));
                *(f32x4*)(x + 4) = *(const f32x4*)(row + (((4 * kk + 2 * h + 1) ^ (r & 7)) << 4));
                if (valid < 32) {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = 16 * kk + 8 * h + e < valid ? x[e] : 0.0f;
                }
            } else {
                const int c = r ^ (h << 5);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = *(const float*)(base + (16 * kk + 8 * h + e) * (GROUPS * 32) + c * 4);
            }
            split(x, p);
        }
    };

    // C tile at (m0, n0), steps [k0, k1) of ceil(k / 32)
    static __device__ __forceinline__ void run(const JvMm& a, int m0, int n0, int k0, int k1, unsigned char* smem, f32x16 (&acc)[MT][NT]) {
        const int w = threadIdx.x >> 6, r31 = threadIdx.x & 31, wm = w % WM, wn = w / WM;
        Side<TA, NA, GA> sa;
        Side<TB, NB, GB> sb;
        sa.init(a.a, a.lda, m0, a.M, a.ca);
        sb.init(a.b, a.ldb, n0, a.N, a.cb);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[m][n][e] = 0.0f;
        // (behind the last step the last one is copied again, into a buffer that nobody reads: the number of copies under way stays the same)
        auto stage = [&](int s) {
            unsigned char* dst = smem + (s - k0) % NS * BUF;
            s = min(s, k1 - 1);
            sa.copy(a.lda, s, TA ? a.ka : a.k, dst);
            sb.copy(a.ldb, s, TB ? a.kb : a.k, dst + GA * GROUP);
        };
#pragma unroll
        for (int i = 0; i < NS - 1; i++) stage(k0 + i);
        for (int s = k0; s < k1; s++) {
            stage(s + NS - 1);
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(AHEAD) : "memory");
            const unsigned char* base = smem + (s - k0) % NS * BUF;
            const int valid = a.k - s * 32;
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                bf16x8 va[MT][3], vb[NT][3];
#pragma unroll
                for (int t = 0; t < MT; t++) sa.read(base, (wm * MT + t) * 32 + r31, kk, valid, va[t]);
#pragma unroll
                for (int t = 0; t < NT; t++) sb.read(base + GA * GROUP, (wn * NT + t) * 32 + r31, kk, valid, vb[t]);
#pragma unroll
                for (int g = 0; g < 6; g++) {
                    const int pa = (0x052 >> (2 * g)) & 3, pb = (0x118 >> (2 * g)) & 3;
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int n = 0; n < NT; n++) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb[n][pb], va[m][pa], acc[m][n], 0, 0, 0);
                }
            }
            // every fragment read of this buffer has returned before any wave stages into it again
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");   // nothing is on its way into LDS any more
    }
    // acc[m][n][e] is C[row(m)][col(n, e)] of the tile, four consecutive e are four consecutive columns
    static __device__ __forceinline__ int row(int m) { return (((threadIdx.x >> 6) % WM) * MT + m) * 32 + (threadIdx.x & 31); }
    static __device__ __forceinline__ int col(int n, int e) {
        return (((threadIdx.x >> 6) / WM) * NT + n) * 32 + (e & 3) + 8 * (e >> 2) + 4 * ((threadIdx.x >> 5) & 1);
    }
};

}  // namespace jvmm
