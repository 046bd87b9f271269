// jv_mm_out.h — matrix products written as they are, on the tiles of jv_mm.h (small) and jv_pipe.h (large).
#pragma once
#include <atomic>

#include "jv_pipe.h"
#include "jv_tile3.h"

namespace jvmm {

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(1))) float f32x1;
typedef __attribute__((ext_vector_type(1))) __bf16 bf16x1;

// a query's target is one of n rows
__device__ __forceinline__ bool known(int target, int64_t n) { return target >= 0 && target < n; }

// the output's rows are 16-B aligned
__host__ __device__ __forceinline__ bool aligned_rows(const JvMmOut& a) { return (uintptr_t)a.out % 16 == 0 && a.ldo % (a.dtype == 0 ? 4 : 8) == 0; }

// Tile L of tm x tn in bands of 8 tiles of A: the 32 workgroups that an XCD runs at a time share 8 tiles of A and 4 of B.
__device__ __forceinline__ void band_order(int L, int tm, int tn, int& m, int& n) {
    const int band = L / (8 * tn), in = L - band * 8 * tn, high = min(8, tm - band * 8);
    n = in / high;
    m = band * 8 + in - n * high;
}

// Lets a kernel have that much LDS, once for each device (a second thread that gets here meanwhile does the same again).
template <auto KERNEL>
static hipError_t lds_of(int bytes) {
    static std::atomic<uint64_t> done[4];   // a bit for each device
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    if (device < 256 && (done[device >> 6].load(std::memory_order_relaxed) >> (device & 63) & 1)) return hipSuccess;
    e = hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && device < 256) done[device >> 6].fetch_or(1ull << (device & 63), std::memory_order_relaxed);
    return e;
}

template <int TY, bool TA, bool TB, bool ENDS>
__global__ __launch_bounds__(512) void jvm_out_pipe_kernel(const JvMmOut a) {
    using P = Pipe<TY, TA, TB, ENDS>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tm = (a.mm.M + P::TM - 1) / P::TM, tn = (a.mm.N + P::TN - 1) / P::TN, tiles = tm * tn;
    const Share share(tiles * a.splits);
    if (!share.mine()) return;
    const int phases = a.mm.kph;
    auto work = [&](int i, Work& w) {
        int L;
        if (!share.at(i, L)) return false;
        int m, n;
        w.part = 0;
        if (a.splits > 1) w.part = L / tiles, L -= w.part * tiles;   // (the tiles of one k range side by side: they share both operands)
        band_order(L, tm, tn, m, n);
        w.m0 = m * P::TM, w.n0 = n * P::TN;
        w.k0 = (int)((int64_t)phases * w.part / a.splits), w.k1 = (int)((int64_t)phases * (w.part + 1) / a.splits);
        return true;
    };
    const float mul = a.norm ? a.mul * *a.norm : a.mul;
    P::run(a.mm, smem, work, [&](const Work& w, f32x16 (&acc)[4][2]) -> int {
        auto value = [&](int m, int n, int e) { return acc[m][n][e] * mul; };
        if (a.dtype != 0) return P::write_bf16(smem, (uint16_t*)a.out, a.ldo, w, a.mm.M, a.mm.N, value);
        return P::write_f32(smem, (float*)a.out + (int64_t)w.part * a.mm.M * a.ldo, a.ldo, a.add, w, a.mm.M, a.mm.N, value);
    });
}

template <int TY, bool TA = false, bool TB = false, bool ENDS = false>
static hipError_t mm_out_pipe(const JvMmOut& a, hipStream_t s) {
    using P = Pipe<TY, TA, TB, ENDS>;
    if (a.mm.M <= 0 || a.mm.N <= 0) return hipSuccess;
    const int64_t all = (int64_t)((a.mm.M + P::TM - 1) / P::TM) * ((a.mm.N + P::TN - 1) / P::TN) * a.splits;
    if (all > 0x7fffffffll || a.splits < 1 || a.splits > a.mm.kph || !aligned_rows(a)) return hipErrorInvalidValue;
    hipError_t e = lds_of<jvm_out_pipe_kernel<TY, TA, TB, ENDS>>(P::LDS);
    if (e != hipSuccess) return e;
    jvm_out_pipe_kernel<TY, TA, TB, ENDS><<<(unsigned)(all < 256 ? (all + 7) / 8 * 8 : 256), P::THREADS, P::LDS, s>>>(a);
    return hipGetLastError();
}

// Tile `i` of `n` when every workgroup has one: those of an XCD (i & 7) take a contiguous run (bijective for any n).
__device__ __forceinline__ int xcd_order(int i, int n) {
    const int xcd = i & 7, slot = i >> 3, q = n >> 3, r = n & 7;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + slot;
}

// A wave's accumulators of 32 rows, turned by way of its own part of LDS (free after T::run), so that a store writes a row's 32 * NT columns one
// behind another: as the lanes hold them, each store would touch 32 rows (dv of 20 x 265 213 x 335, rows not aligned: 285 -> 151 us).
// Piece p (16 B) of row r lies at p ^ (r & 7).
template <class T>
struct Turn {
    static constexpr int COLS = 32 * T::NT;
    static_assert(T::THREADS / 64 * COLS * 128 <= T::LDS);
    const unsigned char* at;
    int r0, c0;   // the tile's row and column of the first element
    __device__ __forceinline__ Turn(unsigned char* smem, int m, const f32x16 (&acc)[T::NT]) {
        const int r31 = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
        unsigned char* to = smem + (threadIdx.x >> 6) * (COLS * 128);
        at = to, r0 = T::row(m) - r31, c0 = T::col(0, 0) - 4 * h;
        asm volatile("" ::: "memory");   // (a wave's LDS accesses are carried out in order: the last rows have been read)
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < T::NT; n++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *(f32x4*)(to + (r31 * (COLS / 4) + ((8 * n + 2 * g + h) ^ (r31 & 7))) * 16) = (f32x4){acc[n][4 * g], acc[n][4 * g + 1], acc[n][4 * g + 2], acc[n][4 * g + 3]};
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
    }
    // the i-th of COLS / (2 W) stores of W columns; `r`, `c`: their place in the tile
    template <class V>
    __device__ __forceinline__ V get(int i, int& r, int& c) const {
        constexpr int W = sizeof(V) / 4;
        const int k = i * 64 + (threadIdx.x & 63), row = k / (COLS / W), col = k % (COLS / W) * W;
        r = r0 + row, c = c0 + col;
        return *(const V*)(at + (row * (COLS / 4) + ((col >> 2) ^ (row & 7))) * 16 + (col & 3) * 4);
    }
};

// workgroup `i` of tiles * splits: one tile over one k range.  TARGETS: JvMmOut.targets is looked at.
template <class T, bool TARGETS = false>
__device__ __forceinline__ void out_tile(const JvMmOut& a, int i, unsigned char* smem) {
    constexpr int MT = T::MT, NT = T::NT;
    const int tm = (a.mm.M + T::TM - 1) / T::TM, tn = (a.mm.N + T::TN - 1) / T::TN, tiles = tm * tn;
    int L = xcd_order(i, tiles * a.splits), part = 0, m0, n0;
    if (a.splits > 1) part = L / tiles, L -= part * tiles;
    band_order(L, tm, tn, m0, n0);
    m0 *= T::TM, n0 *= T::TN;
    const int steps = T::steps(a.mm);
    f32x16 acc[MT][NT];
    T::run(a.mm, m0, n0, (int)((int64_t)steps * part / a.splits), (int)((int64_t)steps * (part + 1) / a.splits), smem, acc);
    const float mul = a.norm ? a.mul * *a.norm : a.mul;
    // elements that every row's start is aligned to: so many a store (scores of 1024 x n x 768, bf16: n = 100 001 220 us, 100 002
    // 203, 100 004 182)
    const uint64_t start = (uint64_t)(uintptr_t)a.out / (a.dtype == 0 ? 4 : 2) | (uint64_t)a.ldo;
    const int64_t slab = (int64_t)part * a.mm.M * a.ldo;
    auto rows = [&](const Turn<T>& turn, auto like, auto half) {   // vectors of as many elements, float32 and bf16
        using V = decltype(like);
        using H = decltype(half);
        constexpr int W = sizeof(V) / 4, stores = Turn<T>::COLS / (2 * W), at_once = stores < 8 ? stores : 8;
#pragma clang loop unroll(disable)
        for (int first = 0; first < stores; first += at_once)
#pragma unroll
        for (int i = first; i < first + at_once; i++) {
            int r, c;
            V v = turn.template get<V>(i, r, c) * mul;
            r += m0, c += n0;
            if (r >= a.mm.M || c >= a.mm.N) continue;
            if (TARGETS && a.targets && !known(a.targets[r], a.n)) v = V{};
            const int64_t at = (int64_t)r * a.ldo + c;
            if (a.dtype == 0) {
                float* p = (float*)a.out + slab + at;
                if (c + W <= a.mm.N) {
                    if (a.add) v += *(const V*)p;
                    *(V*)p = v;
                } else {
#pragma unroll
                    for (int e = 0; e < W; e++)
                        if (c + e < a.mm.N) p[e] = a.add ? p[e] + v[e] : v[e];
                }
            } else {
                __bf16* p = (__bf16*)a.out + at;
                H b;
#pragma unroll
                for (int e = 0; e < W; e++) b[e] = (__bf16)v[e];
                if (c + W <= a.mm.N) {
                    *(H*)p = b;
                } else {
#pragma unroll
                    for (int e = 0; e < W; e++)
                        if (c + e < a.mm.N) p[e] = b[e];
                }
            }
        }
    };
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const Turn<T> turn(smem, m, acc[m]);
        if (start % 4 == 0) rows(turn, f32x4{}, bf16x4{});
        else if (start % 2 == 0) rows(turn, f32x2{}, bf16x2{});
        else rows(turn, f32x1{}, bf16x1{});
    }
}

template <class T>
__global__ __launch_bounds__(T::THREADS, T::RESIDENT) void jvm_out_tile_kernel(const JvMmOut a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    out_tile<T>(a, blockIdx.x, smem);
}

// workgroups of a product on tiles of TM x TN, 0 = none, negative = more than a launch takes
static inline int64_t tile_count(const JvMmOut& a, int TM, int TN, int steps) {
    if (a.mm.M <= 0 || a.mm.N <= 0) return 0;
    if (a.splits < 1 || a.splits > steps || (a.dtype != 0 && a.splits > 1)) return -1;
    const int64_t all = (int64_t)((a.mm.M + TM - 1) / TM) * ((a.mm.N + TN - 1) / TN) * a.splits;
    return all > 0x7fffffffll ? -1 : all;
}

template <class T>
static hipError_t mm_out_tile(const JvMmOut& a, hipStream_t s) {
    const int64_t all = tile_count(a, T::TM, T::TN, T::steps(a.mm));
    if (all <= 0) return all ? hipErrorInvalidValue : hipSuccess;
    hipError_t e = lds_of<jvm_out_tile_kernel<T>>(T::LDS);
    if (e != hipSuccess) return e;
    jvm_out_tile_kernel<T><<<(unsigned)all, T::THREADS, T::LDS, s>>>(a);
    return hipGetLastError();
}

}  // namespace jvmm
