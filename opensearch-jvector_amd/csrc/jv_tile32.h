// jv_tile32.h — the product of jv_mm.h for small shapes whose operands are float32 as they lie in memory.
//
// A float32 product on the bf16 matrix unit: each operand is split into three bf16 parts (x = h + m + l, 24 bits) on the way from LDS into the
// fragments, and the six pairs of parts that reach 2^-24 are multiplied, the smallest first.  Nothing is laid out beforehand: a value is read
// from memory once for each tile that needs it, as 4 bytes, where planes in memory would be written as 6 and read as 12.  k goes by in steps
// of 32; LDS holds NS of them (Tile).  An operand with k along its rows (d components, any number: what lies behind is masked in the last step) is
// staged in 8-row groups of 128 B a row as in Tile; one with k across its rows as 32 rows of TM / TN columns, where the rows 8 .. 15 and
// 24 .. 31 have their 128-B halves of 256 B swapped, so that the two halves of a wave, eight rows apart, read different banks.
// Copies are 16 B a lane from addresses that need 4-B alignment only.  The 16 B that would pass the end of a row start so much earlier that
// they end with it, and their components are taken from so much further back (rows of fewer than four are laid out with four beforehand).
// Bound by the way through a tile's steps and, behind that, by the splitting (704 cycles a step and wave beside 384 of products): loss 64 x 8000 x 384 20 us.
#pragma once
#include "jv_mm.h"

namespace jvmm {

// the six pairs of parts (2,0) (0,2) (1,1) (1,0) (0,1) (0,0), the smallest products first
__device__ __forceinline__ constexpr int part_of_a(int g) { return (0x052 >> (2 * g)) & 3; }
__device__ __forceinline__ constexpr int part_of_b(int g) { return (0x118 >> (2 * g)) & 3; }

// SOLO: one wave (WM = WN = 1) of a workgroup works by itself, in LDS of its own, on every `stride`-th step (KSplit).
template <int MT_, int NT_, int WM, int WN, int NS, bool TA, bool TB, bool SOLO = false>
struct Tile32 {
    using acc_t = f32x16;
    static constexpr bool RAW = true;   // float32 operands as they lie
    static constexpr int MT = MT_, NT = NT_, RESIDENT = 1, E = 16, WIDE = 32 * NT;
    static constexpr int TM = 32 * MT * WM, TN = 32 * NT * WN, WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int GA = TM / 8, GB = TN / 8;                       // KB of a step
    static constexpr int PER = (GA + GB) / WAVES;                        // copies of one wave a step
    static constexpr int BUF = (GA + GB) * GROUP, LDS = NS * BUF;
    static_assert(GA % WAVES == 0 && GB % WAVES == 0, "every wave copies the same number of groups of each operand");
    static_assert((!TA || GA >= 8) && (!TB || GB >= 8), "the swapped halves are 32 columns each");
    static __host__ __device__ __forceinline__ int steps(const JvMm& a) { return (a.k + 31) / 32; }

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

    // four components of a row's last step: those of the 16 B that started earlier from where they are, what lies behind the row as zeros
    static __device__ __forceinline__ f32x4 tail(f32x4 v, int piece, int valid, int k) {
        const int back = k < 4 || 4 * piece >= valid ? 0 : max(4 * piece + 4 - valid, 0);
        if (back & 1) v = (f32x4){v[1], v[2], v[3], v[3]};
        if (back & 2) v = (f32x4){v[2], v[3], v[3], v[3]};
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = 4 * piece + e < valid ? v[e] : 0.0f;
        return v;
    }

    // One operand of `rows` rows of k components (k along) or k rows of `cols` columns (k across); GROUPS * 8 rows or columns from `first` on.
    template <bool ACROSS, int GROUPS>
    struct Side {
        static constexpr int COPIES = GROUPS / WAVES;
        const char* src[COPIES];

        // copy i of this wave is KB number i * WAVES + w: eight rows of 128 B (k along), or rows of GROUPS * 32 B (k across)
        __device__ __forceinline__ void init(const char* base, int64_t ld, int first, int rows, int cols) {
            const int lane = threadIdx.x & 63, w = SOLO ? 0 : threadIdx.x >> 6;
#pragma unroll
            for (int i = 0; i < COPIES; i++) {
                const int c = i * WAVES + w;
                if constexpr (!ACROSS) {
                    src[i] = base + (int64_t)min(first + 8 * c + (lane >> 3), rows - 1) * ld;
                } else {
                    const int byte = c * 1024 + lane * 16, k = byte / (GROUPS * 32);
                    const int col = ((byte % (GROUPS * 32)) >> 2) ^ (((k >> 3) & 1) << 5);
                    src[i] = base + (int64_t)min(first + col, max(cols, 4) - 4) * 4;
                }
            }
        }
        __device__ __forceinline__ void copy(int64_t ld, int step, int k, unsigned char* dst) {
            const int lane = threadIdx.x & 63, w = SOLO ? 0 : threadIdx.x >> 6;
#pragma unroll
            for (int i = 0; i < COPIES; i++) {
                const int c = i * WAVES + w;
                const char* p = src[i];
                if constexpr (!ACROSS) p += (int64_t)min(step * 32 + (((lane & 7) ^ (lane >> 3)) << 2), max(k, 4) - 4) * 4;
                else p += (int64_t)min(step * 32 + (c * 1024 + lane * 16) / (GROUPS * 32), k - 1) * ld;
                glds16(p, dst + c * (ACROSS ? 1024 : GROUP));
            }
        }
        // where column r of the tile lies in a row of the step (k across)
        static __device__ __forceinline__ int place(int r, int first, int cols) {
            const int back = cols < 4 ? 0 : min(max(first + (r & ~3) + 4 - cols, 0), 3);
            return (r & ~3) + min((r & 3) + back, 3);
        }
        // eight k's (16 kk + 8 h ..) of row r, or of the column at `r` (place); LAST: the step has `valid` of 32 components, `k` in all (k along)
        template <bool LAST>
        static __device__ __forceinline__ void read(const unsigned char* base, int r, int kk, int valid, int k, bf16x8 (&p)[3]) {
            const int h = (threadIdx.x >> 5) & 1;
            float x[8];
            if constexpr (!ACROSS) {
                const unsigned char* row = base + (r >> 3) * GROUP + (r & 7) * 128;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int piece = 4 * kk + 2 * h + half;
                    f32x4 v = *(const f32x4*)(row + ((piece ^ (r & 7)) << 4));
                    if constexpr (LAST) v = tail(v, piece, valid, k);
#pragma unroll
                    for (int e = 0; e < 4; e++) x[4 * half + e] = v[e];
                }
            } else {
                const int c = r ^ (h << 5);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = *(const float*)(base + (16 * kk + 8 * h + e) * (GROUPS * 32) + c * 4);
            }
            split(x, p);
        }
    };

    // one step
    template <bool LAST>
    static __device__ __forceinline__ void multiply(const JvMm& a, const unsigned char* base, const int (&ra)[MT], const int (&rb)[NT], int valid, f32x16 (&acc)[MT][NT]) {
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            bf16x8 va[MT][3], vb[NT][3];
#pragma unroll
            for (int t = 0; t < MT; t++) Side<TA, GA>::template read<LAST>(base, ra[t], kk, valid, a.k, va[t]);
#pragma unroll
            for (int t = 0; t < NT; t++) Side<TB, GB>::template read<LAST>(base + GA * GROUP, rb[t], kk, valid, a.k, vb[t]);
#pragma unroll
            for (int g = 0; g < 6; g++) {
                const int pa = part_of_a(g), pb = part_of_b(g);
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int n = 0; n < NT; n++) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb[n][pb], va[m][pa], acc[m][n], 0, 0, 0);
            }
        }
    }
    // C tile at (m0, n0), steps [k0, k1) of ceil(k / 32)
    static __device__ __forceinline__ void run(const JvMm& a, int m0, int n0, int k0, int k1, unsigned char* smem, f32x16 (&acc)[MT][NT], int stride = 1) {
        const int w = SOLO ? 0 : threadIdx.x >> 6, r31 = threadIdx.x & 31, wm = w % WM, wn = w / WM;
        Side<TA, GA> sa;
        Side<TB, GB> sb;
        sa.init(a.a, a.lda, m0, a.M, a.ca);
        sb.init(a.b, a.ldb, n0, a.N, a.cb);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[m][n][e] = 0.0f;
        int ra[MT], rb[NT];
#pragma unroll
        for (int t = 0; t < MT; t++) ra[t] = (wm * MT + t) * 32 + r31, ra[t] = TA ? sa.place(ra[t], m0, a.ca) : ra[t];
#pragma unroll
        for (int t = 0; t < NT; t++) rb[t] = (wn * NT + t) * 32 + r31, rb[t] = TB ? sb.place(rb[t], n0, a.cb) : rb[t];
        auto stage = [&](int s, int to) {
            unsigned char* dst = smem + to * BUF;
            sa.copy(a.lda, s, TA ? a.ka : a.k, dst);
            sb.copy(a.ldb, s, TB ? a.kb : a.k, dst + GA * GROUP);
        };
#pragma unroll
        for (int i = 0; i < NS - 1; i++)
            if (k0 + i * stride < k1) stage(k0 + i * stride, i);
        int buf = 0;
        for (int s = k0; s < k1; s += stride) {
            if (s + (NS - 1) * stride < k1) stage(s + (NS - 1) * stride, buf == 0 ? NS - 1 : buf - 1);
            wait_step<NS, PER, SOLO>(SOLO ? (k1 - 1 - s) / stride : k1 - 1 - s);
            const unsigned char* base = smem + buf * BUF;
            if ((s + 1) * 32 <= a.k) multiply<false>(a, base, ra, rb, 32, acc);
            else multiply<true>(a, base, ra, rb, a.k - s * 32, acc);   // (apart: the masks would cost every step a third more)
            release_step<SOLO>();
            buf = buf + 1 == NS ? 0 : buf + 1;
        }
    }
    // acc[m][n][e] is C[row(m)][col(n, e)] of the tile, four consecutive e are four consecutive columns
    static __device__ __forceinline__ int row(int m) { return (((threadIdx.x >> 6) % WM) * MT + m) * 32 + (threadIdx.x & 31); }
    static __device__ __forceinline__ int col(int n, int e) {
        return (((threadIdx.x >> 6) / WM) * NT + n) * 32 + (e & 3) + 8 * (e >> 2) + 4 * ((threadIdx.x >> 5) & 1);
    }
};

// A 32 x 32 tile whose k steps four waves share, each with its own LDS and no barrier between steps; wave w ends up with 8 of the 32 columns.
// For few tiles with a long k, where the way through one tile's steps is what counts.
template <class Solo>
struct KSplit {
    using acc_t = f32x4;
    static constexpr bool RAW = true;   // float32 operands as they lie
    static constexpr int MT = 1, NT = 1, RESIDENT = 1, E = 4, WIDE = 8, TM = 32, TN = 32, THREADS = 256, LDS = 4 * Solo::LDS;
    static __host__ __device__ __forceinline__ int steps(const JvMm& a) { return Solo::steps(a); }
    static __device__ __forceinline__ void run(const JvMm& a, int m0, int n0, int k0, int k1, unsigned char* smem, f32x4 (&acc)[1][1]) {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        f32x16 mine[1][1];
        Solo::run(a, m0, n0, k0 + w, k1, smem + w * Solo::LDS, mine, 4);
        __syncthreads();
        f32x4* sh = (f32x4*)smem;   // [wave][four values][lane]
#pragma unroll
        for (int g = 0; g < 4; g++) sh[(w * 4 + g) * 64 + lane] = (f32x4){mine[0][0][4 * g], mine[0][0][4 * g + 1], mine[0][0][4 * g + 2], mine[0][0][4 * g + 3]};
        __syncthreads();
        acc[0][0] = (sh[w * 64 + lane] + sh[(4 + w) * 64 + lane]) + (sh[(8 + w) * 64 + lane] + sh[(12 + w) * 64 + lane]);
        __syncthreads();
    }
    static __device__ __forceinline__ int row(int) { return threadIdx.x & 31; }
    static __device__ __forceinline__ int col(int, int e) { return (threadIdx.x >> 6) * 8 + 4 * ((threadIdx.x >> 5) & 1) + e; }
};

}  // namespace jvmm
