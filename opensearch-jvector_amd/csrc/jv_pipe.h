// jv_pipe.h — the matrix product of jv_mm.h for large shapes: 256 x 256 tiles, eight waves in two groups that take turns.
//
// A resident workgroup of 512 threads walks a list of tiles; k goes by in PHASES of 64 bytes a row.  Four regions of LDS hold the phases
// in flight (32 KB each, copied straight from global memory three phases ahead), and the copies never pause: behind a tile's last
// phases they are the next tile's first.  Waves w and w + 4 share a SIMD and belong to different groups; group 1 is half a phase behind:
//
//     group 0:   read q | multiply q | read q+1 | multiply q+1 | ...
//     group 1:          | read q     | multiply q | read q+1   | ...        ( | = barrier )
//
// so one of them feeds the SIMD's matrix unit while the other reads its fragments.  With barriers counted from group 0's first (B0), phase q
// is read by group 0 before B(2q) and by group 1 before B(2q+1); every wave waits for its own copies of phase q before B(2q-1), and the
// copies into the region of phase q-1 are issued in phase q's read, behind B(2q-1): nothing is overwritten before both groups read it.
//
// An operand lies either with k along its rows (its row index is a row or column of C) or, bf16 only, with k across them (TA / TB: its rows
// are k, as a gradient's operands lie).  k along rows: a row's 64 bytes are four 16-B pieces, piece p at p ^ ((row >> 2) & 3), so a
// fragment read's 16 consecutive rows cover the 64 banks once.  k across rows: 32 rows of 256 columns, read through the transposing
// LDS read (16 lanes give four rows of 16 and take 16 columns of four); piece p of row k at p ^ ((k & 3) << 2), so four rows cover the banks.
// Bound by the matrix unit: 8192^3 in bf16 1277 TFLOP/s (a library's product: 1423), at the 1.6 - 1.8 GHz that power leaves; tiles of 1024 components
// with an epilogue each 1000 - 1075.  Four waves of 128 x 128 each, which read a third less from LDS, were slower.
#pragma once
#include "jv_mm.h"

namespace jvmm {

struct Work {
    int m0, n0;      // first row and column of the tile
    int k0, k1;      // phases of the kph in all
    int part;        // which k range
};

// ENDS: JvMm.tail_b is there (looking for it costs 1 % otherwise).
template <int TY, bool TA = false, bool TB = false, bool ENDS = false>
struct Pipe {
    using acc_t = f32x16;
    static constexpr bool RAW = false;
    static constexpr int E = 16, WIDE = 64;
    static constexpr int MT = 4, NT = 2, TM = 256, TN = 256, THREADS = 512;   // waves: 2 along M, 4 along N
    static constexpr int REGION = 32768, SCALES = 4 * REGION, SCRATCH = SCALES + (TY == BF16 ? 0 : 2 * 8192);
    static constexpr int LDS = SCRATCH + 4 * 4096;   // 4 KB for waves w and w + 4: they are never in their epilogue at the same time
    static_assert(TY == BF16 || (!TA && !TB), "8-bit operands have k along their rows");
    static_assert(TB || !ENDS);

    template <int N>
    static __device__ __forceinline__ void wait_copies() {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    }
    // copies of the next phase have landed: eight younger ones may be under way, and in the two phases behind an epilogue its stores too
    static __device__ __forceinline__ void wait_next(int stores) {
        if (stores == 16) wait_copies<24>();
        else if (stores == 32) wait_copies<40>();
        else wait_copies<8>();
    }
    static __device__ __forceinline__ void barrier() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
    // what this lane holds: acc[m][n][e] is C[row(m)][col(n, e)] of the tile, four consecutive e are four consecutive columns
    static __device__ __forceinline__ int row(int m) { return ((threadIdx.x >> 6) & 1) * 128 + m * 32 + (threadIdx.x & 31); }
    static __device__ __forceinline__ int col(int n, int e) {
        return (threadIdx.x >> 7) * 64 + n * 32 + (e & 3) + 8 * (e >> 2) + 4 * ((threadIdx.x >> 5) & 1);
    }

    // `work(i, w)`: the i-th tile of this workgroup, false (and w untouched) behind the last; the first always exists.  `done(w, acc)`: what
    // becomes of it; returns how many stores every wave has issued for certain (0, 16 or 32).
    template <class NextWork, class Done>
    static __device__ __forceinline__ void run(const JvMm& a, unsigned char* smem, NextWork&& work, Done&& done) {
        const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int group = w >> 2;
        const int wm = w & 1, wn = w >> 1, h = lane >> 5, r31 = lane & 31;

        // ---- copies: two of A and two of B for each wave and phase ----
        Work sw;
        work(0, sw);
        int si = 0, sk = sw.k0, sreg = 0;
        const char *pa[2], *pb[2];   // k along rows: the row's piece; k across: the column's piece of row 0
        bool ends = false;           // k across: this piece is the last of B's row
        auto rows = [&]() {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                // k along rows: lane l of a copy fills row l >> 2, piece l & 3 of 16 rows; k across: row l >> 5, piece l & 31 of two
                if constexpr (!TA) pa[i] = a.a + (int64_t)min(sw.m0 + 16 * (i * 8 + w) + (lane >> 2), a.M - 1) * a.lda + ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
                else pa[i] = a.a + (int64_t)min(sw.m0 + 8 * ((lane & 31) ^ (((2 * w + (lane >> 5)) & 3) << 2)), a.ca - 8) * 2;
                if constexpr (!TB) pb[i] = a.b + (int64_t)min(sw.n0 + 16 * (i * 8 + w) + (lane >> 2), a.N - 1) * a.ldb + ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
                else {
                    const int col = min(sw.n0 + 8 * ((lane & 31) ^ (((2 * w + (lane >> 5)) & 3) << 2)), a.cb - 8);
                    pb[i] = a.b + (int64_t)col * 2, ends = ENDS && col == a.cb - 8;
                }
            }
        };
        rows();
        const int64_t end_b = a.end_b - 16 - ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
        auto stage = [&]() {
            const int64_t off = (int64_t)sk * 64;
            unsigned char* dst = smem + sreg * REGION + w * 1024;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int k = sk * 32 + 16 * i + 2 * w + (lane >> 5);
                glds16(pa[i] + (TA ? (int64_t)min(k, a.ka - 1) * a.lda : off), dst + i * 8192);
                const char* p = pb[i] + (TB ? (int64_t)min(k, a.kb - 1) * a.ldb : min(off, end_b));
                if (ENDS && ends && k >= a.kb - 1) p = a.tail_b;
                glds16(p, dst + 16384 + i * 8192);
            }
            sreg = (sreg + 1) & 3;
            if (++sk == sw.k1) {   // on to the next tile (behind the last: the same one again, never read)
                if (work(si + 1, sw)) si++;
                sk = sw.k0;
                rows();
            }
        };
        stage();
        stage();
        stage();

        // ---- fragments ----
        // k along rows: the two 16-B pieces of a lane and phase: bf16 k 8 (2j + h) .. + 7; e4m3 (F8) 32 h .. + 31, (F8W) 16 (2j + h) .. + 15
        const int x = (r31 >> 2) & 3;
        const int o0 = ((TY == F8 ? 2 * h : h) ^ x) << 4, o1 = ((TY == F8 ? 2 * h + 1 : 2 + h) ^ x) << 4;
        // k across rows: rows 16 j + 8 h + 4 half + (0 .. 3), columns 32 t + 16 (lane bit 4) + (0 .. 15)
        const int tk = (lane & 15) >> 2;
        auto across = [&](const unsigned char* base, int first, int j) -> i32x4 {   // 32 columns from `first` on
            const int c = first + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
            const unsigned char* p = base + (16 * j + 8 * h + tk) * 512 + (((c >> 3) ^ (tk << 2)) << 4) + (c & 4) * 2;
            return __builtin_bit_cast(i32x4, __builtin_shufflevector(read_across(p), read_across(p + 4 * 512), 0, 1, 2, 3, 4, 5, 6, 7));
        };

        // ---- scales: thread t keeps row t of the two tiles; a window of 16 blocks (32 phases) goes from global memory to LDS while the one
        //      before it is multiplied, and a fragment's rows are read from there four blocks at a time ----
        uint32_t sca[MT], scb[NT], raw[4];
        int back = 0;   // bytes that this row's window starts behind what was read: nothing is read behind the matrix (16 blocks at least in all)
        auto load_scales = [&](const Work& at, int block) {
            if constexpr (TY != BF16) {
                const bool isb = tid >= 256;
                const int rows = isb ? a.N : a.M, row = min((isb ? at.n0 - 256 : at.m0) + tid, rows - 1);
                const int nk = a.kph >> 1;
                const int64_t want = (int64_t)row * nk + block, end = (int64_t)rows * nk - 16, from = want < end ? want : end;
                __builtin_memcpy(raw, (isb ? a.sb : a.sa) + from, 16);
                back = (int)(want - from);
            }
        };
        auto keep_scales = [&](int window) {
            if constexpr (TY != BF16) {
                const int by = back & 3, words = back >> 2;
                uint32_t v[4];
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = __builtin_amdgcn_alignbyte(i < 3 ? raw[i + 1] : 0, raw[i], by);
                if (words & 1) v[0] = v[1], v[1] = v[2], v[2] = v[3];
                if (words & 2) v[0] = v[2], v[1] = v[3];
                *(i32x4*)(smem + SCALES + (window & 1) * 8192 + tid * 16) = (i32x4){(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
            }
        };
        auto take_scales = [&](int window, int block) {
            if constexpr (TY != BF16) {
                const unsigned char* p = smem + SCALES + (window & 1) * 8192 + (block & 12);
#pragma unroll
                for (int t = 0; t < MT; t++) sca[t] = *(const uint32_t*)(p + ((wm * MT + t) * 32 + r31) * 16);
#pragma unroll
                for (int t = 0; t < NT; t++) scb[t] = *(const uint32_t*)(p + (256 + (wn * NT + t) * 32 + r31) * 16);
            }
        };

        Work cw;
        work(0, cw);
        load_scales(cw, 0);
        keep_scales(0);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        barrier();
        if (group) barrier();
        int reg = 0, window = 0, stores = 0;
        for (int i = 0;; i++) {
            Work nw = cw;
            const bool more = work(i + 1, nw);
            f32x16 acc[MT][NT];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[m][n][e] = 0.0f;
            const int phases = cw.k1 - cw.k0;
            for (int q = 0; q < phases; q++) {
                const unsigned char* base = smem + reg * REGION;
                i32x4 fa[MT][2], fb[NT][2];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if constexpr (TB) {
                        fb[t][0] = across(base + 16384, (wn * NT + t) * 32, 0), fb[t][1] = across(base + 16384, (wn * NT + t) * 32, 1);
                    } else {
                        const unsigned char* p = base + 16384 + ((wn * NT + t) * 32 + r31) * 64;
                        fb[t][0] = *(const i32x4*)(p + o0), fb[t][1] = *(const i32x4*)(p + o1);
                    }
                }
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    if constexpr (TA) {
                        fa[t][0] = across(base, (wm * MT + t) * 32, 0), fa[t][1] = across(base, (wm * MT + t) * 32, 1);
                    } else {
                        const unsigned char* p = base + ((wm * MT + t) * 32 + r31) * 64;
                        fa[t][0] = *(const i32x4*)(p + o0), fa[t][1] = *(const i32x4*)(p + o1);
                    }
                }
                reg = (reg + 1) & 3;
                if constexpr (TY != BF16) {
                    if ((q & 7) == 0) take_scales(window, q >> 1);
                    if ((q & 31) == 0) load_scales(q + 32 < phases ? cw : nw, q + 32 < phases ? (q >> 1) + 16 : 0);
                    if ((q & 31) == 31 || q + 1 == phases) keep_scales(++window);
                }
                stage();
                if (group) wait_next(q < 2 ? stores : 0);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                barrier();
                __builtin_amdgcn_s_setprio(1);
                if constexpr (TY == BF16) {
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int m = 0; m < MT; m++)
#pragma unroll
                            for (int n = 0; n < NT; n++)
                                acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fb[n][j]), __builtin_bit_cast(bf16x8, fa[m][j]), acc[m][n], 0, 0, 0);
                } else if constexpr (TY == F8) {
                    const int sh = ((q >> 1) & 3) * 8;
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int n = 0; n < NT; n++)
                            acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                                __builtin_shufflevector(fb[n][0], fb[n][1], 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(fa[m][0], fa[m][1], 0, 1, 2, 3, 4, 5, 6, 7),
                                acc[m][n], 0, 0, 0, (int)(scb[n] >> sh), 0, (int)(sca[m] >> sh));
                } else {
                    const int sh = ((q >> 1) & 3) * 8;
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            bf16x8 va[MT], vb[NT];
#pragma unroll
                            for (int n = 0; n < NT; n++) vb[n] = widen(fb[n][j][2 * half], fb[n][j][2 * half + 1], (int)(scb[n] >> sh) & 255);
#pragma unroll
                            for (int m = 0; m < MT; m++) {
                                va[m] = widen(fa[m][j][2 * half], fa[m][j][2 * half + 1], (int)(sca[m] >> sh) & 255);
#pragma unroll
                                for (int n = 0; n < NT; n++) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb[n], va[m], acc[m][n], 0, 0, 0);
                            }
                        }
                }
                // (the products stay on this side of the barrier)
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int n = 0; n < NT; n++) asm volatile("" : "+v"(acc[m][n]));
                __builtin_amdgcn_s_setprio(0);
                if (!group) wait_next(q < 2 ? stores : 0);
                if (q + 1 < phases) barrier();
            }
            stores = done(cw, acc);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the scratch changes hands)
            barrier();
            if (!more) break;
            cw = nw;
        }
        if (!group) barrier();
        wait_copies<0>();   // the copies behind the last tile have landed before LDS changes hands
        __syncthreads();
    }

    // threadIdx.x, computed anew: an epilogue's addresses would otherwise be kept through the whole product, whose registers are all taken
    // (scores of 256 x 500 000 x 128: 155 and 133 us).
    static __device__ __forceinline__ int own_thread() {
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
        return t;
    }

    // Writes a tile whose elements are value(m, n, e) as rows of float32 or bf16, `ldo` elements apart, rows < M and columns < N; the rows
    // are 16-B aligned.  They go through LDS, so that a store writes whole 128-B lines: 32 rows of 128 B at a time, piece p of row r at
    // p ^ ((r >> 1) & 7).  (Other rows go to the small tiles: element by element from here, scores of 256 x 500 001 x 768 took 496 us, there 343.)
    // Returns the stores that every wave has issued.
    template <class V>
    static __device__ __forceinline__ int write_bf16(unsigned char* smem, uint16_t* out, int64_t ldo, const Work& at, int M, int N, V&& value) {
        const int tid = own_thread(), lane = tid & 63, w = tid >> 6, h = lane >> 5, r31 = lane & 31;
        const int m0 = at.m0 + (w & 1) * 128, n0 = at.n0 + (w >> 1) * 64;
        unsigned char* sc = smem + SCRATCH + (w & 3) * 4096;
        const bool full = at.m0 + TM <= M && at.n0 + TN <= N;
#pragma unroll
        for (int m = 0; m < MT; m++) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    bf16x4 v;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = (__bf16)value(m, n, 4 * g + e);
                    *(bf16x4*)(sc + r31 * 128 + (((4 * n + g) ^ ((r31 >> 1) & 7)) << 4) + 8 * h) = v;
                }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = i * 8 + (lane >> 3);
                const i32x4 v = *(const i32x4*)(sc + r * 128 + (((lane & 7) ^ ((r >> 1) & 7)) << 4));
                const int gr = m0 + m * 32 + r, gc = n0 + (lane & 7) * 8;
                uint16_t* p = out + (int64_t)gr * ldo + gc;
                if (full || (gr < M && gc + 8 <= N)) {
                    *(i32x4*)p = v;
                } else if (gr < M) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (gc + e < N) p[e] = (uint16_t)((uint32_t)v[e >> 1] >> (16 * (e & 1)));
                }
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
        }
        return full ? 16 : 0;
    }
    template <class V>
    static __device__ __forceinline__ int write_f32(unsigned char* smem, float* out, int64_t ldo, bool add, const Work& at, int M, int N, V&& value) {
        const int tid = own_thread(), lane = tid & 63, w = tid >> 6, h = lane >> 5, r31 = lane & 31;
        const int m0 = at.m0 + (w & 1) * 128, n0 = at.n0 + (w >> 1) * 64;
        unsigned char* sc = smem + SCRATCH + (w & 3) * 4096;
        const bool full = at.m0 + TM <= M && at.n0 + TN <= N;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = value(m, n, 4 * g + e);
                    *(f32x4*)(sc + r31 * 128 + (((2 * g + h) ^ ((r31 >> 1) & 7)) << 4)) = v;
                }
                __builtin_amdgcn_wave_barrier();
                asm volatile("" ::: "memory");
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = i * 8 + (lane >> 3);
                    f32x4 v = *(const f32x4*)(sc + r * 128 + (((lane & 7) ^ ((r >> 1) & 7)) << 4));
                    const int gr = m0 + m * 32 + r, gc = n0 + n * 32 + (lane & 7) * 4;
                    float* p = out + (int64_t)gr * ldo + gc;
                    if (full || (gr < M && gc + 4 <= N)) {
                        if (add) v += *(const f32x4*)p;
                        *(f32x4*)p = v;
                    } else if (gr < M) {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (gc + e < N) p[e] = add ? p[e] + v[e] : v[e];
                    }
                }
                __builtin_amdgcn_wave_barrier();
                asm volatile("" ::: "memory");
            }
        return full && !add ? 32 : 0;
    }
};

// The tiles of one launch: the workgroups of one XCD (blockIdx & 7 of a grid of a multiple of 8) take a contiguous run of the `all` tiles.
struct Share {
    int first, count, slot, step;
    __device__ __forceinline__ explicit Share(int all) {
        const int xcd = blockIdx.x & 7, q = all >> 3, r = all & 7;
        first = xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q;
        count = q + (xcd < r ? 1 : 0);
        slot = blockIdx.x >> 3;
        step = gridDim.x >> 3;
    }
    __device__ __forceinline__ bool mine() const { return slot < count; }
    __device__ __forceinline__ bool at(int i, int& tile) const {
        if (slot + i * step >= count) return false;
        tile = first + slot + i * step;
        return true;
    }
};

}  // namespace jvmm
