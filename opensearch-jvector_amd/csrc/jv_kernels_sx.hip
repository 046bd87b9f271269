// jv_kernels_sx.hip — softmax cross entropy of queries over all rows of an index without keeping the logits, and its gradient, which keeps a weight in the place
// of each, a piece of the rows at a time (gfx950).
//
//   z_ij = scale q_i . v_j     lse_i = log sum_j exp z_ij     loss_i = lse_i - z_i,t(i) = log(1 + sum_(j != t(i)) exp(z_ij - z_i,t(i)))
//   g_ij = w_i scale (exp(z_ij - lse_i) - [j = t(i)])         dq_i = sum_j g_ij v_j         dv_j = sum_i g_ij q_i
// The sums leave the target out, and g at the target is w_i scale (exp(-loss_i) - 1) where the losses are given: a learnt pair's loss and gradient have all the
// digits of float32 products, not those that are left behind a 1.
//
// Forward: a workgroup walks tiles of rows for one panel of queries, and every lane keeps the running maximum and sum of ITS rows (one column of
// the accumulators is one query: no exchange until the end); the workgroups' partials are joined by a second kernel.  Backward: the logits
// are computed again, a piece of the rows at a time, and written once as g [query][row]; dq reads g with k along its rows, dv with k across
// them (the transposing LDS read), so nothing is transposed in memory.  Logarithms and exponentials are base 2 inside (c = scale log2 e).
//
// bf16 operands are multiplied as they are (products exact in float32, float32 sums); g is rounded to bf16 once: half a step, 2^-8 relative, for
// each term of a sum over rows or queries, the size of the gradient's own final rounding.  The entry at a query's target is the one term that
// stands alone: what it lacks (`rest`) is added to dq in float32.  float32 operands and g are three bf16 parts (24 bits) and a product is the six
// pairs of them that reach 2^-24: float32's accuracy at 1.5 times the rate of its own matrix instruction (1423 / 6 against 154 TFLOP/s).
//
// What bounds it (MI355X; a large copy moves 4.7 TB/s, a large bf16 product runs at 1423 TFLOP/s):
//   few queries (bf16 300, float32 100: as many operations as a byte of rows pays for): the rows' bytes.  Loss 256 x 1 000 000 x 768 bf16: 450 us,
//     3.4 TB/s and 870 TFLOP/s, near both; loss 11 x 257 776 x 1272 float32: 268 us, 4.9 TB/s.
//   many queries: the matrix unit, and behind each tile the exponentials (a quarter of the rate of other instructions), which no product runs
//     beside.  Step 4096 x 131 072 x 1024 bf16: 4.17 ms, 1055 TFLOP/s over its four products; float32 777 x 30 011 x 381: 550 us, 775 TFLOP/s.
//   little of everything: the launches.  Step 32 x 1000 x 64 float32: 37 us for five.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "jv_mm.h"
#include "jv_mm_out.h"

using namespace jvmm;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }
// v_mul_legacy_f32: 0 where one of them is, also beside NaN and infinity (the compiler has it as an intrinsic without a builtin)
__device__ float times_or_0(float x, float w) __asm("llvm.amdgcn.fmul.legacy");

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
// what has to be laid out: rows as padded bf16 planes [rows][planes][kp], and what the gradient needs of each query
// ---------------------------------------------------------------------------------------------
// A query without a target (jvmm::known) takes no part in the gradients, whatever it (a batch's padding may be NaN) or a row holds: its row of g is zeros, and so
// are its row among dv's operands and its own gradient.
template <typename T>
__device__ __forceinline__ void pack(const JvSxPrepare& a, const JvSxPrepare::Matrix& m, int64_t first, int64_t step) {   // eight components a thread
    constexpr int P = sizeof(T) == 4 ? 3 : 1;
    const int d = a.d, kp = m.kp, per = kp / 8;
    auto dead = [&](int64_t r) { return m.clean && !known(a.targets[r], a.n); };
    if (m.raw) {
        for (int64_t i = first; i < m.rows * kp; i += step) {
            const int64_t r = i / kp;
            const int c = (int)(i - r * kp);
            ((float*)m.out)[i] = c < d && !dead(r) ? (float)((const T*)m.x)[r * m.stride + c] : 0.0f;
        }
        return;
    }
    for (int64_t i = first; i < m.rows * per; i += step) {
        const int64_t r = i < 0x100000000ll ? (int64_t)((uint32_t)i / (uint32_t)per) : i / per;
        const int at = (int)(i - r * per) * 8;
        const T* row = (const T*)m.x + r * m.stride;
        T x[8];
        if (dead(r)) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = (T)0.0f;
        } else if (at + 8 <= d) {
            __builtin_memcpy(x, row + at, sizeof(x));   // (no alignment is asked for)
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int c = m.shift && at < d ? d - 8 + e : at + e;
                x[e] = c >= at && c < d ? row[c] : (T)0.0f;
            }
        }
        uint16_t p[3][8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (P == 1) {
                p[0][e] = __builtin_bit_cast(uint16_t, x[e]);
            } else {
                uint16_t q[3];
                planes3(x[e], q);
#pragma unroll
                for (int k = 0; k < 3; k++) p[k][e] = q[k];
            }
        }
#pragma unroll
        for (int k = 0; k < P; k++) {
            i32x4 o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (int)((uint32_t)p[k][2 * e] | ((uint32_t)p[k][2 * e + 1] << 16));
            *(i32x4*)((uint16_t*)m.out + (r * P + k) * kp + at) = o;
        }
    }
}

// `unit`: what the weights are divided by.  `loss` (nullptr: not known): g at the target is w (exp(-loss) - 1), with all the digits that the loss has; from lse,
// p - 1 is left with what a float32 lse leaves of it (half a step of 20 is 1e-6).
__device__ __forceinline__ JvSxQuery query_of(const float* lse, const float* loss, const float* w, const int32_t* targets, int64_t n, int i, float unit) {
    const int t = targets[i];
    if (!known(t, n)) return {__builtin_inff(), 0.0f, -1, 0.0f};
    const float w0 = w ? w[i] : 1.0f, lse2 = lse[i] * 1.44269504088896341f;
    // no probabilities (a logit was NaN or +inf, or all of them -inf): NaN shows, also beside a weight of 0 (times_or_0)
    if (!(lse[i] > -__builtin_inff()) || w0 != w0) return {__builtin_nanf(""), __builtin_nanf(""), t, __builtin_nanf("")};
    // lse log2(e) - lse2: what both roundings left out, up to 2^-19 for a logarithm of 40 and as much of p
    const float lacks = fabsf(lse2) < __builtin_inff() ? fmaf(lse[i], 1.44269504088896341f, -lse2) + lse[i] * 1.92596299112661747e-8f : 0.0f;
    return {lse2, w0 * exp2_(-lacks) / unit, t, loss ? w0 / unit * expm1f(-loss[i]) : w0 / unit};
}

// The weights are divided by the largest of them (`norm`, multiplied back in float32 at the end): an entry of g at a target is then just
// below 1 for the largest weight, where bf16's step is finest in relation.  Every workgroup finds the largest anew: no
// more than 64 of them.
__device__ __forceinline__ void queries(const JvSxPrepare& a, int part, int parts) {
    __shared__ float tops[4];
    float top = 0.0f;
    if (a.w) {
#pragma unroll 8
        for (int i = threadIdx.x; i < a.nq; i += 256) {
            const int t = a.targets[i];
            const float w = a.w[i];
            if (known(t, a.n)) top = fmaxf(top, fabsf(w));
        }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    // (no weights, none but zeros, or one that is not finite: 1, so that what is not finite shows in the gradient)
    const float unit = a.w && top > 0.0f && top < __builtin_inff() ? top : 1.0f;
    int i = part * 256 + threadIdx.x;
    if (i == 0) *a.norm = unit;
    if (a.last && i < 8) ((__bf16*)a.tail)[i] = a.d / 8 * 8 + i < a.d ? ((const __bf16*)a.last)[a.d / 8 * 8 + i] : (__bf16)0.0f;
    for (; i < a.nq; i += parts * 256) {
        a.query[i] = query_of(a.lse, a.loss, a.w, a.targets, a.n, i, unit);
        a.rest[i] = 0.0f;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void jvs_prepare_kernel(const JvSxPrepare a, int g0, int g1, int g2) {   // workgroups for the matrices, the rest for the queries
    int i = blockIdx.x;
    if (i < g0) return pack<T>(a, a.m[0], (int64_t)i * 256 + threadIdx.x, (int64_t)g0 * 256);
    i -= g0;
    if (i < g1) return pack<T>(a, a.m[1], (int64_t)i * 256 + threadIdx.x, (int64_t)g1 * 256);
    i -= g1;
    if (i < g2) return pack<T>(a, a.m[2], (int64_t)i * 256 + threadIdx.x, (int64_t)g2 * 256);
    queries(a, i - g2, gridDim.x - g0 - g1 - g2);
}
extern "C" hipError_t jvk_sx_prepare(const JvSxPrepare* a, hipStream_t s) {
    int g[3];
    for (int k = 0; k < 3; k++) g[k] = (int)std::min<int64_t>((a->m[k].rows * std::max(a->m[k].kp / 8, 1) + 255) / 256, 32768);
    const unsigned grid = (unsigned)(g[0] + g[1] + g[2] + (a->query ? std::min((a->nq + 255) / 256, 64) : 0));
    if (grid == 0) return hipSuccess;
    if (a->dtype == 0) jvs_prepare_kernel<float><<<grid, 256, 0, s>>>(*a, g[0], g[1], g[2]);
    else jvs_prepare_kernel<__bf16><<<grid, 256, 0, s>>>(*a, g[0], g[1], g[2]);
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

// A lane's part of a tile: MT queries, NT * 16 rows each.  `rows`: how many rows the tile has in all.  Four instructions a logit: the maximum, the
// scaled difference (c <= 0: the smallest product is the largest logit), the exponential, the sum.
// `m0`, `n0`: where the tile lies.  The target's own product is kept apart (`hit`) and left out of the maximum and the sum: where a pair is learnt its
// term would be the 1 that all other terms together, which are the loss, are rounded against.
template <class Core, int MT, int NT>
__device__ __forceinline__ void add_tile(const JvSxLoss& a, typename Core::acc_t (&acc)[MT][NT], int m0, int n0, const int (&want)[MT], float (&top)[MT], float (&sum)[MT]) {
    const float c = a.c;
    const int rows = a.mm.N - n0;
    const int first = Core::col(0, 0) & ~(Core::WIDE < 32 ? 7 : 31);   // this wave's columns
    const float none = c < 0.0f ? __builtin_inff() : -__builtin_inff();   // (the target and what is behind the last row: the logit is -inf)
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int at = want[m] - n0;
        if (__any(at >= first && at < first + Core::WIDE)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < Core::E; e++)
                    if (Core::col(n, e) == at) a.hit[m0 + Core::row(m)] = acc[m][n][e], acc[m][n][e] = none;
        }
    }
    if (rows < Core::TN) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < Core::E; e++) acc[m][n][e] = Core::col(n, e) < rows ? acc[m][n][e] : none;
    }
    float best[MT];
    if (c < 0.0f) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
            best[m] = none;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < Core::E; e++) best[m] = fminf(best[m], acc[m][n][e]);
        }
    } else {
#pragma unroll
        for (int m = 0; m < MT; m++) {
            best[m] = none;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < Core::E; e++) best[m] = fmaxf(best[m], acc[m][n][e]);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; m++) {
        // (c = 0: a lane that has rows has 0 for its maximum)
        const float now = fmaxf(top[m], best[m] == none ? -__builtin_inff() : best[m] * c), ref = now == -__builtin_inff() ? 0.0f : now;
        float s = sum[m] * exp2_(top[m] - ref);
        if (c == 0.0f) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < Core::E; e++) {   // (by their places: -inf may be a product, and 0 times that is NaN)
                    const int col = Core::col(n, e);
                    s += col < rows && col != want[m] - n0 ? exp2_(acc[m][n][e] * 0.0f) : 0.0f;
                }
        } else {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < Core::E; e++) s += exp2_(fmaf(acc[m][n][e], c, -ref));
        }
        top[m] = now;
        sum[m] = s;
    }
}

// the piece's row that is query `q`'s target, -1 if there is none
__device__ __forceinline__ int wanted(const JvSxLoss& a, int q) {
    const int64_t at = q < a.mm.M && a.targets ? a.targets[q] - a.row0 : -1;
    return at >= 0 && at < a.mm.N ? (int)at : -1;
}

// joins what the lanes and waves of a workgroup hold of the same queries and writes one partial for each of the panel's queries
template <int TM, int MT, int WN, class Row>
__device__ __forceinline__ void write_partials(const JvSxLoss& a, unsigned char* smem, int m0, int split, int wn, Row&& row, float (&top)[MT], float (&sum)[MT]) {
    float* sh = (float*)smem;   // [WN][TM][2]
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; m++) {
        join(top[m], sum[m], __shfl_xor(top[m], 32, 64), __shfl_xor(sum[m], 32, 64));
        if ((threadIdx.x & 63) < 32) {
            sh[(wn * TM + row(m)) * 2] = top[m];
            sh[(wn * TM + row(m)) * 2 + 1] = sum[m];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TM; i += blockDim.x) {
        if (m0 + i >= a.mm.M) continue;
        float m = sh[i * 2], s = sh[i * 2 + 1];
#pragma unroll
        for (int k = 1; k < WN; k++) join(m, s, sh[(k * TM + i) * 2], sh[(k * TM + i) * 2 + 1]);
        float2* p = a.part + (int64_t)(m0 + i) * a.splits + split;
        if (!a.first) join(m, s, p->x, p->y);
        *p = make_float2(m, s);
    }
}

__global__ __launch_bounds__(512) void jvs_loss_pipe_kernel(const JvSxLoss a) {
    using P = Pipe<BF16>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    // one panel of queries and every `splits`-th tile of rows; the panels of a split side by side: they share its rows
    const int panels = (a.mm.M + P::TM - 1) / P::TM, tiles = (a.mm.N + P::TN - 1) / P::TN;
    const Share share(panels * a.splits);
    int L;
    if (!share.at(0, L)) return;
    const int split = L / panels, m0 = (L - split * panels) * P::TM;
    float top[4], sum[4];
    int want[4];
#pragma unroll
    for (int m = 0; m < 4; m++) top[m] = -__builtin_inff(), sum[m] = 0.0f, want[m] = wanted(a, m0 + P::row(m));
    if (split < tiles)
        P::run(
            a.mm, smem,
            [&](int i, Work& w) {
                const int t = split + i * a.splits;
                if (t >= tiles) return false;
                w.m0 = m0, w.n0 = t * P::TN, w.k0 = 0, w.k1 = a.mm.kph;
                return true;
            },
            [&](const Work& w, f32x16 (&acc)[4][2]) -> int {
                add_tile<P>(a, acc, w.m0, w.n0, want, top, sum);
                return 0;
            });
    write_partials<P::TM, 4, 4>(a, smem, m0, split, threadIdx.x >> 7, [](int m) { return P::row(m); }, top, sum);
}

template <class T, int WM, int WN>
__global__ __launch_bounds__(T::THREADS, T::RESIDENT) void jvs_loss_tile_kernel(const JvSxLoss a) {
    constexpr int MT = T::MT, NT = T::NT;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int panels = (a.mm.M + T::TM - 1) / T::TM, tiles = (a.mm.N + T::TN - 1) / T::TN;
    const Share share(panels * a.splits);
    int L;
    if (!share.at(0, L)) return;
    const int split = L / panels, m0 = (L - split * panels) * T::TM;
    float top[MT], sum[MT];
    int want[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) top[m] = -__builtin_inff(), sum[m] = 0.0f, want[m] = wanted(a, m0 + T::row(m));
    for (int t = split; t < tiles; t += a.splits) {
        typename T::acc_t acc[MT][NT];
        T::run(a.mm, m0, t * T::TN, 0, T::steps(a.mm), smem, acc);
        add_tile<T>(a, acc, m0, t * T::TN, want, top, sum);
    }
    write_partials<T::TM, MT, WN>(a, smem, m0, split, (threadIdx.x >> 6) / WM, [](int m) { return T::row(m); }, top, sum);
}

// bf16: the large tiles where they fill the chip and more than half of one is queries.  float32: everything as it lies where that is no more than
// one tile of 128 x 128 a CU (laying out costs a launch), the queries as planes above (step 777 x 30 011 x 381: 555 us; with both operands as
// planes on the large tiles, every pair of planes a pass over k: 695 us; step 2000 x 30 000 x 1024: 2.82 and 2.90 ms).
extern "C" int jvk_sx_path(int nq, int64_t rows, int f32) {
    if (!f32) return nq > 128 && ((nq + 255) / 256) * ((rows + 255) / 256) >= 192 ? JV_SX_LARGE : JV_SX_TILES;
    return (int64_t)((nq + 127) / 128) * ((rows + 127) / 128) <= 256 ? JV_SX_RAW : JV_SX_PLANES;
}

// Queries and rows of the smaller tiles: 32 x 128 and 64 x 128 (float32 also 96 x 128) for up to so many queries, the rows being streamed and as
// little as possible multiplied for nothing; 128 x 128 otherwise; but where that is no more than one tile a CU 64 x 64, with four steps of k
// under way: the way to memory and the multiplications of one tile's steps are what counts then (float32, 118 x 18 x 843: 66 -> 36 us).
// float32 with no more than four tiles of 32 x 32 a CU and at least eight steps of k: those, four waves sharing a tile's steps, two steps of
// each wave under way where there is more than one tile a CU and four otherwise (a step of 28 x 46 x 1167: 90 -> 43 us, of 100 x 2000 x 768: 80 -> 49;
// a loss of 256 x 2000 x 768: 32 -> 20, of 16 x 30 000 x 768: 34 -> 29; of 512 x 4000 x 768, eight tiles a CU: 43 and 47; bf16, a fifth of the
// instructions a step: 54 and 54).
struct Shape {
    int m, n;
    bool few;
};
static int64_t tiles32(int nq, int64_t rows) { return (int64_t)((nq + 31) / 32) * ((rows + 31) / 32); }
static Shape shape_of(int path, int nq, int64_t rows, int d) {
    if (path == JV_SX_LARGE) return {256, 256, false};
    if (path == JV_SX_RAW && d > 7 * 32 && tiles32(nq, rows) <= 1024) return {32, 32, true};
    const bool few = (int64_t)((nq + 127) / 128) * ((rows + 127) / 128) <= 256;
    if (path == JV_SX_PLANES) return {nq > 96 ? 128 : (nq + 31) / 32 * 32, 128, false};
    if (nq <= 32) return {32, 128, few};
    if (few) return {64, 64, true};
    return {nq <= 64 ? 64 : 128, 128, false};
}

// Workgroups that share a panel of 256 queries: as many as make up whole rounds of the 256 CUs, each of them walking as many of the tiles and
// costing about one more to begin.
static int large_splits(int nq, int64_t rows) {
    const int64_t panels = std::max((nq + 255) / 256, 1), tiles = std::max<int64_t>((rows + 255) / 256, 1);
    int64_t best = 1, least = INT64_MAX;
    for (int rounds = 1; rounds <= 8; rounds++) {
        const int64_t s = std::min(std::max<int64_t>(256 * rounds / panels, 1), tiles), cost = (panels * s + 255) / 256 * ((tiles + s - 1) / s + 1);
        if (cost < least) best = s, least = cost;
    }
    return (int)best;
}

// (two or three workgroups a CU with the small tiles)
extern "C" int jvk_sx_loss_splits(int path, int nq, int64_t rows, int d) {
    const Shape t = shape_of(path, nq, rows, d);
    if (path == JV_SX_LARGE) return large_splits(nq, rows);
    const int full = t.n == 32 ? 512 : t.m == 128 || t.n == 64 || path == JV_SX_PLANES ? 512 : 768;
    const int64_t panels = std::max((nq + t.m - 1) / t.m, 1), tiles = std::max<int64_t>((rows + t.n - 1) / t.n, 1);
    return (int)std::min(std::max<int64_t>(full / panels, 1), tiles);
}

template <class T, int WM, int WN>
static hipError_t loss_tile(const JvSxLoss& a, hipStream_t s) {
    hipError_t e = lds_of<jvs_loss_tile_kernel<T, WM, WN>>(T::LDS);
    if (e != hipSuccess) return e;
    const int64_t all = (int64_t)((a.mm.M + T::TM - 1) / T::TM) * a.splits;
    if (all > 0x7ffffff0ll) return hipErrorInvalidValue;
    jvs_loss_tile_kernel<T, WM, WN><<<(unsigned)((all + 7) / 8 * 8), T::THREADS, T::LDS, s>>>(a);
    return hipGetLastError();
}
extern "C" hipError_t jvk_sx_loss(const JvSxLoss* a, hipStream_t s) {
    using P = Pipe<BF16>;
    if (a->mm.N <= 0 || a->mm.M <= 0) return hipSuccess;
    if (a->splits < 1) return hipErrorInvalidValue;
    const Shape t = shape_of(a->path, a->mm.M, a->mm.N, a->mm.k);
    if (t.n == 32) return tiles32(a->mm.M, a->mm.N) <= 256 ? loss_tile<KSplit<Tile32<1, 1, 1, 1, 4, false, false, true>>, 1, 4>(*a, s) : loss_tile<KSplit<Tile32<1, 1, 1, 1, 2, false, false, true>>, 1, 4>(*a, s);
    if (a->path == JV_SX_RAW) return t.m == 32 ? loss_tile<Tile32<1, 1, 1, 4, 4, false, false>, 1, 4>(*a, s) : loss_tile<Tile32<1, 1, 2, 2, 4, false, false>, 2, 2>(*a, s);
    if (a->path == JV_SX_PLANES) {
        if (t.m == 32) return loss_tile<Tile3<1, false, false>, 1, 4>(*a, s);
        if (t.m == 64) return loss_tile<Tile3<2, false, false>, 1, 4>(*a, s);
        return t.m == 96 ? loss_tile<Tile3<3, false, false>, 1, 4>(*a, s) : loss_tile<Tile3<4, false, false>, 1, 4>(*a, s);
    }
    if (a->path == JV_SX_TILES) {
        if (t.m == 128) return loss_tile<Tile<BF16, 2, 2, 2, 2, 2>, 2, 2>(*a, s);
        if (t.n == 64) return loss_tile<Tile<BF16, 1, 1, 2, 2, 4>, 2, 2>(*a, s);
        if (t.m == 64) return loss_tile<Tile<BF16, 2, 1, 1, 4, 2>, 1, 4>(*a, s);
        return t.few ? loss_tile<Tile<BF16, 1, 1, 1, 4, 4>, 1, 4>(*a, s) : loss_tile<Tile<BF16, 1, 1, 1, 4, 2>, 1, 4>(*a, s);
    }
    hipError_t e = lds_of<jvs_loss_pipe_kernel>(P::LDS);
    if (e != hipSuccess) return e;
    const int64_t all = (int64_t)((a->mm.M + P::TM - 1) / P::TM) * a->splits;
    if (all > 0x7ffffff0ll) return hipErrorInvalidValue;
    jvs_loss_pipe_kernel<<<(unsigned)((all + 7) / 8 * 8), P::THREADS, P::LDS, s>>>(*a);
    return hipGetLastError();
}

// One wave a query: join the partials, which are o = log sum_(j not the target) exp z_j; with the target's logit z
//   loss = log(1 + exp(o - z)),   lse = z + loss,
// each as the larger of the two and log1p of what is behind it.  The few operations behind the sums are in 64 bits: as float32 o and z would be rounded
// by 2e-6 near 40, and a loss near 0, exp(o - z), by that share of itself.
__global__ __launch_bounds__(256) void jvs_join_kernel(const float2* __restrict__ part, int splits, int nq, float c, const float* __restrict__ hit,
                                                       const int32_t* __restrict__ targets, int64_t n, float* __restrict__ loss, float* __restrict__ lse) {
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (i >= nq) return;
    float m = -__builtin_inff(), s = 0.0f;
#pragma unroll 4
    for (int k = lane; k < splits; k += 64) {
        const float2 p = part[(int64_t)i * splits + k];
        join(m, s, p.x, p.y);
    }
    for (int off = 32; off >= 1; off >>= 1) join(m, s, __shfl_xor(m, off, 64), __shfl_xor(s, off, 64));
    if (lane != 0) return;
    constexpr double ln2 = 0.69314718055994530942, inf = __builtin_inf();
    const double rest = (double)m * ln2 + log((double)s);
    double all = rest, own = 0.0;
    if (targets && known(targets[i], n)) {
        const double z = (double)hit[i] * c * ln2;
        if (z == -inf) {   // probability 0
            own = rest - z;
        } else {           // (an infinite logit leaves no probabilities)
            const double behind = log1p(exp(-fabs(rest - z))), none = z == inf ? z - z : 0.0;
            all = (rest > z ? rest : z) + behind + none;
            own = (rest > z ? rest - z : 0.0) + behind + none;
        }
    }
    lse[i] = (float)all;
    loss[i] = (float)own;
}

extern "C" hipError_t jvk_sx_join(const float2* part, int splits, int nq, float c, const float* hit, const int32_t* targets, int64_t n, float* loss, float* lse,
                                  hipStream_t s) {
    if (nq <= 0) return hipSuccess;
    jvs_join_kernel<<<(nq + 3) / 4, 256, 0, s>>>(part, splits, nq, c, hit, targets, n, loss, lse);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------
// backward: the logits again, as weights g
// ---------------------------------------------------------------------------------------------
// g of a lane's columns of one query, in place of the logits; `cols`: how many of the tile's columns are rows of the piece; `hit`: the target's
// column; `told`: the losses are known.  Three instructions a value; the target, which few tiles hold, and the last tile's end are seen to apart.
template <class Core, int NT>
__device__ __forceinline__ void weigh(typename Core::acc_t (&acc)[NT], const JvSxQuery& q, float c, int cols, int hit, bool told, bool lossy, float* rest) {
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < Core::E; e++) acc[n][e] = times_or_0(exp2_(fmaf(acc[n][e], c, -q.lse2)), q.w);   // (no target: 0)
    const int first = Core::col(0, 0) & ~(Core::WIDE < 32 ? 7 : 31);   // this wave's columns
    if (__any(hit >= first && hit < first + Core::WIDE)) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < Core::E; e++)
                if (Core::col(n, e) == hit) {
                    acc[n][e] = told ? q.own : acc[n][e] - q.own;
                    if (lossy) *rest = acc[n][e] - (float)(__bf16)acc[n][e];   // (one lane holds it; three planes lack nothing)
                }
    }
    if (cols < Core::TN) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < Core::E; e++) acc[n][e] = Core::col(n, e) < cols ? acc[n][e] : 0.0f;
    }
}

// One panel of queries and every `splits`-th tile of rows a workgroup, as in the forward pass: what it needs of its queries stays in registers
// (loaded behind each tile, it would wait for the copies under way: adapter 256 x 400 000 x 128, 231 -> 215 us; step 4096 x 131 072 x 1024, 4.22 -> 4.14 ms).
__global__ __launch_bounds__(512) void jvs_weights_kernel(const JvSxWeights a, int splits) {
    using P = Pipe<BF16>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int panels = (a.mm.M + P::TM - 1) / P::TM, tiles = (a.mm.N + P::TN - 1) / P::TN;
    const Share share(panels * splits);
    int L;
    if (!share.at(0, L)) return;
    const int split = L / panels, m0 = (L - split * panels) * P::TM;
    const int padded = (a.mm.M + 63) / 64 * 64;
    JvSxQuery q[4];
    int at[4];
#pragma unroll
    for (int m = 0; m < 4; m++) {
        const int r = m0 + P::row(m);
        q[m] = {__builtin_inff(), 0.0f, -1, 0.0f};
        if (r < a.mm.M) q[m] = a.query[r];
        const int64_t t = q[m].target - a.row0;
        at[m] = q[m].target >= 0 && t >= 0 && t < a.mm.N ? (int)t : -1;
    }
    if (split >= tiles) return;
    P::run(
        a.mm, smem,
        [&](int i, Work& w) {
            const int t = split + i * splits;
            if (t >= tiles) return false;
            w.m0 = m0, w.n0 = t * P::TN, w.k0 = 0, w.k1 = a.mm.kph;
            return true;
        },
        [&](const Work& w, f32x16 (&acc)[4][2]) -> int {
#pragma unroll
            for (int m = 0; m < 4; m++) weigh<P>(acc[m], q[m], a.c, a.mm.N - w.n0, at[m] - w.n0, a.loss, true, a.rest + w.m0 + P::row(m));
            return P::write_bf16(smem, (uint16_t*)a.g, a.kv, w, padded, a.kv, [&](int m, int n, int e) { return acc[m][n][e]; });
        });
}

// Rows of G: the queries and, where they are no whole steps of the product that has them for k, a row of zeros, which that product reads as
// all the rows behind it.
static __host__ __device__ __forceinline__ int padded_queries(const JvSxWeights& a) {
    const int step = a.path == JV_SX_RAW || a.path == JV_SX_PLANES ? 32 : 64;
    return a.mm.M % step ? a.mm.M + 1 : a.mm.M;
}

constexpr int CLEANED = 2048;   // values that a workgroup copies

// the same on small tiles, one a workgroup
template <class T>
__global__ __launch_bounds__(T::THREADS, T::RESIDENT) void jvs_weights_tile_kernel(const JvSxWeights a) {
    constexpr int MT = T::MT, NT = T::NT;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int padded = padded_queries(a), tm = (padded + T::TM - 1) / T::TM, tn = (a.kv + T::TN - 1) / T::TN;
    const int copies = gridDim.x - tm * tn;   // workgroups that copy the queries for dv, the first ones: short beside a tile's
    if constexpr (T::RAW) {
        if ((int)blockIdx.x < copies) {
            const uint32_t d = a.mm.k, all = (uint32_t)a.mm.M * d;
#pragma unroll
            for (int k = 0; k < CLEANED / 256; k++) {
                const uint32_t i = blockIdx.x * CLEANED + k * 256 + threadIdx.x, r = i / d;
                if (i < all) a.clean[i] = known(a.targets[r], a.n) ? *((const float*)(a.mm.a + r * a.mm.lda) + (i - r * d)) : 0.0f;
            }
            return;
        }
    }
    int m0, n0;
    band_order(xcd_order(blockIdx.x - copies, tm * tn), tm, tn, m0, n0);
    m0 *= T::TM, n0 *= T::TN;
    typename T::acc_t acc[MT][NT];
    T::run(a.mm, m0, n0, 0, T::steps(a.mm), smem, acc);
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int r = m0 + T::row(m);
        JvSxQuery q = {__builtin_inff(), 0.0f, -1, 0.0f};
        if (r < a.mm.M) q = a.query ? a.query[r] : query_of(a.lse, a.loss, a.w, a.targets, a.n, r, 1.0f);
        weigh<T>(acc[m], q, a.c, a.mm.N - n0, q.target >= 0 ? (int)(q.target - a.row0) - n0 : -1, a.loss, a.path == JV_SX_TILES, a.rest + r);
        // (kv is a multiple of 64: four columns are in or out together)
        auto put = [&](int r, int c, f32x4 v) {
            if (r >= padded || c >= a.kv) return;
            if (a.path == JV_SX_RAW) {
                *(f32x4*)((float*)a.g + (int64_t)r * a.kv + c) = v;
                return;
            }
            const int planes = a.path == JV_SX_PLANES ? 3 : 1;
            uint16_t* p = (uint16_t*)a.g + (int64_t)r * planes * a.kv + c;
            for (int k = 0; k < planes; k++, p += a.kv) {
                const bf16x4 b = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
                *(bf16x4*)p = b;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] -= (float)b[e];
            }
        };
        if constexpr (T::E == 4) {
            put(r, n0 + T::col(0, 0), acc[m][0]);
        } else {
            const Turn<T> turn(smem, m, acc[m]);
#pragma unroll
            for (int i = 0; i < Turn<T>::COLS / 8; i++) {
                int tr, tc;
                const f32x4 v = turn.template get<f32x4>(i, tr, tc);
                put(m0 + tr, n0 + tc, v);
            }
        }
    }
}

template <class T>
static hipError_t weights_tile(const JvSxWeights& a, hipStream_t s) {
    const int64_t all = (int64_t)((padded_queries(a) + T::TM - 1) / T::TM) * ((a.kv + T::TN - 1) / T::TN);
    const int64_t extra = a.clean ? ((int64_t)a.mm.M * a.mm.k + CLEANED - 1) / CLEANED : 0;
    if (all + extra > 0x7fffffffll || extra * CLEANED > 0xffffffffll) return hipErrorInvalidValue;   // (256 tiles of 128 x 128 have 2^15 queries at most)
    hipError_t e = lds_of<jvs_weights_tile_kernel<T>>(T::LDS);
    if (e != hipSuccess) return e;
    jvs_weights_tile_kernel<T><<<(unsigned)(all + extra), T::THREADS, T::LDS, s>>>(a);
    return hipGetLastError();
}

extern "C" hipError_t jvk_sx_weights(const JvSxWeights* a, hipStream_t s) {
    using P = Pipe<BF16>;
    if (a->mm.M <= 0 || a->mm.N <= 0) return hipSuccess;
    const Shape t = shape_of(a->path, a->mm.M, a->mm.N, a->mm.k);
    if (t.n == 32) return tiles32(a->mm.M, a->mm.N) <= 256 ? weights_tile<KSplit<Tile32<1, 1, 1, 1, 4, false, false, true>>>(*a, s) : weights_tile<KSplit<Tile32<1, 1, 1, 1, 2, false, false, true>>>(*a, s);
    if (a->path == JV_SX_RAW) return weights_tile<Tile32<1, 1, 2, 2, 4, false, false>>(*a, s);
    if (a->path == JV_SX_PLANES) {
        if (t.m == 32) return weights_tile<Tile3<1, false, false>>(*a, s);
        if (t.m == 64) return weights_tile<Tile3<2, false, false>>(*a, s);
        return t.m == 96 ? weights_tile<Tile3<3, false, false>>(*a, s) : weights_tile<Tile3<4, false, false>>(*a, s);
    }
    if (a->path == JV_SX_TILES) {
        // (up to 31 queries: 64 rows of G would be half empty; adapter 19 x 556 840 x 128: 109 -> 100 us)
        if (padded_queries(*a) <= 32) return t.few ? weights_tile<Tile<BF16, 1, 1, 1, 4, 4>>(*a, s) : weights_tile<Tile<BF16, 1, 1, 1, 4, 2>>(*a, s);
        if (t.few) return weights_tile<Tile<BF16, 1, 1, 2, 2, 4>>(*a, s);
        return t.m == 128 ? weights_tile<Tile<BF16, 2, 2, 2, 2, 2>>(*a, s) : weights_tile<Tile<BF16, 2, 1, 1, 4, 2>>(*a, s);
    }
    const int splits = large_splits(a->mm.M, a->mm.N);
    const int64_t all = (int64_t)((a->mm.M + P::TM - 1) / P::TM) * splits;
    if (all > 0x7ffffff0ll) return hipErrorInvalidValue;
    hipError_t e = lds_of<jvs_weights_kernel>(P::LDS);
    if (e != hipSuccess) return e;
    jvs_weights_kernel<<<(unsigned)((all + 7) / 8 * 8), P::THREADS, P::LDS, s>>>(*a, splits);
    return hipGetLastError();
}

// dq = G V: G's rows are queries, V's rows are k.  dv = G^T Q: the rows of both are k.  On small tiles both share a launch.
template <class TQ, class TV>
__global__ __launch_bounds__(256) void jvs_grads_tile_kernel(const JvMmOut q, const JvMmOut v, int first) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    if ((int)blockIdx.x < first) out_tile<TQ, true>(q, blockIdx.x, smem);
    else out_tile<TV>(v, blockIdx.x - first, smem);
}
template <class TQ, class TV>
static hipError_t grads_tile(const JvMmOut* q, const JvMmOut* v, hipStream_t s) {
    static_assert(TQ::LDS == TV::LDS && TQ::THREADS == 256 && TV::THREADS == 256);
    const int64_t nq = q ? tile_count(*q, TQ::TM, TQ::TN, TQ::steps(q->mm)) : 0, nv = v ? tile_count(*v, TV::TM, TV::TN, TV::steps(v->mm)) : 0;
    if (nq < 0 || nv < 0 || nq + nv > 0x7fffffffll) return hipErrorInvalidValue;
    if (nq + nv == 0) return hipSuccess;
    hipError_t e = lds_of<jvs_grads_tile_kernel<TQ, TV>>(TQ::LDS);
    if (e != hipSuccess) return e;
    jvs_grads_tile_kernel<TQ, TV><<<(unsigned)(nq + nv), 256, TQ::LDS, s>>>(q ? *q : JvMmOut{}, v ? *v : JvMmOut{}, (int)nq);
    return hipGetLastError();
}

// The gradients' products have d columns: with up to 128 half a large tile would be multiplied for nothing.
static int grads_path(int path, int d) { return path == JV_SX_LARGE && d <= 128 ? JV_SX_TILES : path; }

// k ranges of a gradient of `rows` rows: once around the CUs with the large tiles, twice with the small ones; at least four and eight steps in
// each.  (dv, `across`, step 4096 x 4096 x 768, bf16: 104 us of one range, 40 of five.)
extern "C" int jvk_sx_grad_splits(int path, int64_t rows, int d, int64_t k, int across) {
    path = grads_path(path, d);
    const bool large = path == JV_SX_LARGE;
    const bool few = path == JV_SX_RAW && !across && rows <= 64;
    const int tm = large ? 256 : few ? 64 : path == JV_SX_PLANES && !across ? shape_of(path, (int)rows, k, 0).m : 128, tn = large ? 256 : few ? 64 : 128;
    const int64_t tiles = std::max<int64_t>((rows + tm - 1) / tm, 1) * ((d + tn - 1) / tn);
    const int64_t steps = path == JV_SX_RAW || path == JV_SX_PLANES ? (k + 31) / 32 : (k + 63) / 64;
    return (int)std::max<int64_t>(std::min<int64_t>((large ? 256 : 512) / tiles, steps / (large ? 4 : 8)), 1);
}
extern "C" hipError_t jvk_sx_grads(const JvMmOut* q, const JvMmOut* v, int path, hipStream_t s) {
    path = grads_path(path, q ? q->mm.N : v->mm.N);
    hipError_t e = hipSuccess;
    if (path == JV_SX_LARGE) {
        if (q) e = q->mm.tail_b ? mm_out_pipe<BF16, false, true, true>(*q, s) : mm_out_pipe<BF16, false, true>(*q, s);
        if (v && e == hipSuccess) e = aligned_rows(*v) ? mm_out_pipe<BF16, true, true>(*v, s) : mm_out_tile<Tile<BF16, 2, 2, 2, 2, 2, true, true>>(*v, s);
        return e;
    }
    if (path == JV_SX_PLANES) {
        if (q) {
            const int m = shape_of(path, q->mm.M, 0, 0).m;
            e = m == 32 ? mm_out_tile<Tile3<1, false, true>>(*q, s) : m == 64 ? mm_out_tile<Tile3<2, false, true>>(*q, s) : m == 96 ? mm_out_tile<Tile3<3, false, true>>(*q, s) : mm_out_tile<Tile3<4, false, true>>(*q, s);
        }
        if (v && e == hipSuccess) e = mm_out_tile<Tile3<4, true, true>>(*v, s);
        return e;
    }
    // 64 x 64 where 128 x 128 would be no more than one tile a CU; in float32, whose operands are split for every tile, for dq of up to 64 queries too
    // (adapter 43 x 13 015 x 1296: 131 -> 122 us; bf16: 2 % either way)
    int64_t tiles = 0;
    for (const JvMmOut* o : {q, v})
        if (o) tiles += (int64_t)((o->mm.M + 127) / 128) * ((o->mm.N + 127) / 128) * o->splits;
    if (path == JV_SX_RAW) {
        using Q64 = Tile32<1, 1, 2, 2, 4, false, true>;
        using V128 = Tile32<2, 2, 2, 2, 2, true, true>;
        if (tiles <= 256) return grads_tile<Q64, Tile32<1, 1, 2, 2, 4, true, true>>(q, v, s);
        return q && q->mm.M <= 64 ? grads_tile<Q64, V128>(q, v, s) : grads_tile<Tile32<2, 2, 2, 2, 2, false, true>, V128>(q, v, s);
    }
    if (tiles <= 256) return grads_tile<Tile<BF16, 1, 1, 2, 2, 4, false, true>, Tile<BF16, 1, 1, 2, 2, 4, true, true>>(q, v, s);
    return grads_tile<Tile<BF16, 2, 2, 2, 2, 2, false, true>, Tile<BF16, 2, 2, 2, 2, 2, true, true>>(q, v, s);
}

// partial sums -> the queries' gradient, and what G lacked at the target.  A row's columns, four a lane, are shared by 256 / G lanes, its partial
// sums by G lanes, which are joined in a fixed order: with few columns and hundreds of partial sums the way through one lane's sums is
// what counts (64 x 32 of 512 partial sums: 31 us with G = 1, 4 with 16).
template <typename T, int G>
__global__ __launch_bounds__(256) void jvs_finish_kernel(const JvSxFinish q, const JvSxFinish v, int d, int64_t lds, float mul, const float* __restrict__ norm) {
    constexpr int L = 256 / G;
    __shared__ f32x4 part[G > 1 ? 256 : 1];
    const bool second = blockIdx.x >= q.rows;
    const JvSxFinish& a = second ? v : q;
    const int64_t r = second ? blockIdx.x - q.rows : blockIdx.x;
    const int g = threadIdx.x / L, c = ((int)threadIdx.x % L + (int)blockIdx.y * L) * 4;   // (lds is a multiple of 64)
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < d) {
        const float* p = a.slab + r * lds + c;
#pragma unroll 8
        for (int k = g; k < a.splits; k += G) x += *(const f32x4*)(p + k * a.rows * lds);
    }
    if constexpr (G > 1) {
        part[threadIdx.x] = x;
        __syncthreads();
        if (g > 0) return;
#pragma unroll
        for (int k = 1; k < G; k++) x += part[k * L + threadIdx.x];
    }
    const float by = norm ? mul * *norm : mul, lack = a.rest ? a.rest[r] : 0.0f;
    const T* target = lack != 0.0f ? (const T*)a.vectors + a.query[r].target * a.v_stride : nullptr;
    T* out = (T*)a.out + r * a.ldo;
    const bool dead = a.targets && !known(a.targets[r], a.n);   // (0 times a row that is not finite)
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (c + e < d) out[c + e] = (T)(dead ? 0.0f : (lack != 0.0f ? fmaf(lack, (float)target[c + e], x[e]) : x[e]) * by);
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
extern "C" hipError_t jvk_sx_finish(const JvSxFinish* q, const JvSxFinish* v, int d, int64_t lds, float mul, const float* norm, int dtype, hipStream_t s) {
    const int64_t rows = (q ? q->rows : 0) + (v ? v->rows : 0);
    if (rows <= 0 || d <= 0) return hipSuccess;
    if (rows > 0x7fffffffll) return hipErrorInvalidValue;
    const int splits = std::max(q ? q->splits : 1, v ? v->splits : 1), groups = splits >= 32 ? 16 : splits >= 4 ? 4 : 1, lanes = 256 / groups;
    const dim3 grid((unsigned)rows, (unsigned)((d + 4 * lanes - 1) / (4 * lanes)));
    auto run = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(q ? *q : JvSxFinish{}, v ? *v : JvSxFinish{}, d, lds, mul, norm); };
    if (dtype == 0) run(groups == 16 ? jvs_finish_kernel<float, 16> : groups == 4 ? jvs_finish_kernel<float, 4> : jvs_finish_kernel<float, 1>);
    else run(groups == 16 ? jvs_finish_kernel<__bf16, 16> : groups == 4 ? jvs_finish_kernel<__bf16, 4> : jvs_finish_kernel<__bf16, 1>);
    return hipGetLastError();
}
extern "C" hipError_t jvk_sx_fill(void* out, int dtype, int64_t stride, int64_t rows, int d, float value, hipStream_t s) {
    if (rows <= 0 || d <= 0) return hipSuccess;
    if (dtype == 0) jvs_fill_kernel<float><<<grid_for(rows * d), 256, 0, s>>>((float*)out, stride, rows, d, value);
    else jvs_fill_kernel<__bf16><<<grid_for(rows * d), 256, 0, s>>>((__bf16*)out, stride, rows, d, value);
    return hipGetLastError();
}
