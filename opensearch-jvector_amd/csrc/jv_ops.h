// jv_ops.h — argument blocks of the training and 8-bit scoring kernels (jv_kernels_f8.hip, jv_kernels_sx.hip), shared with jv_abi_ops.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// One product of rows with rows, C[i][j] = sum_k A[i][k] B[j][k]: both operands as rows of whole 128-B steps (64 bf16 or 128 e4m3),
// 16-B aligned.  A float32 operand is three bf16 planes side by side in its row (x = h + m + l, 24 bits); its product is the six
// plane pairs that reach 2^-24, walked as six segments of the same k range, the smallest first.
struct JvMm {
    const char *a, *b;
    int64_t lda, ldb;      // bytes from row to row
    int32_t M, N;          // rows of A / of B
    int32_t nk;            // 128-B steps of one segment
    int32_t segs;          // 1 (bf16, e4m3) or 6 (float32)
    const uint8_t *sa, *sb;  // e4m3: scale bytes [M][nk] / [N][nk]
};

// the logits' forward pass: A = vectors, B = queries
struct JvSxLoss {
    JvMm mm;
    float c;               // scale * log2(e)
    int32_t splits;        // workgroups that share a query panel's rows
    float* part;           // [2][splits][N]: maxima, then sums (log2 domain)
    int32_t first;         // partials of an earlier piece of the rows are in `part` already: 0 = join them
};
// one piece of the gradient's weights: G = w scale (p - [j = t]) as bf16 planes, by query and by row
struct JvSxWeights {
    JvMm mm;               // A = vectors of this piece, B = queries
    float c, scale;
    int64_t row0;          // first row of this piece
    const float* lse;      // [N] natural log
    const float* w;        // [N] or nullptr = 1
    const int32_t* targets;
    int64_t n;             // rows in all (a target outside [0, n) is none)
    int32_t planes;        // 1 or 3
    uint16_t* g;           // [N][planes][kv]  (nullptr: not asked for)
    uint16_t* gt;          // [M][planes][kq]
    int32_t kv, kq;        // columns padded to 64, the padding written as zeros
};
// a product written as it is
struct JvMmOut {
    JvMm mm;
    int32_t dtype;         // JV_DTYPE_*
    void* out;             // [M][ldo]
    int64_t ldo;           // elements
    int32_t splits;        // > 1 or slab != nullptr: partial sums over k ranges, float32 [splits][M][N]
    float* slab;
    int32_t add;           // slab: add to what is there
};

// sets jv_last_error() and returns `code` (jv_abi.cpp)
__attribute__((visibility("hidden"))) int jvi_fail(int code, const char* fmt, ...);

extern "C" {
hipError_t jvk_f8_encode(const void* x, int dtype, int64_t stride, int64_t n, int d, uint8_t* codes, uint8_t* scales, hipStream_t s);
hipError_t jvk_f8_decode(const uint8_t* codes, const uint8_t* scales, int64_t n, int d, void* x, int dtype, int64_t stride, hipStream_t s);
hipError_t jvk_f8_score(const JvMmOut* a, hipStream_t s);

hipError_t jvk_sx_pack(const void* x, int dtype, int64_t stride, int64_t rows, int d, int kp, uint16_t* out, hipStream_t s);
hipError_t jvk_sx_pack_t(const void* x, int dtype, int64_t stride, int rows, int d, int kr, uint16_t* out, hipStream_t s);
hipError_t jvk_sx_loss(const JvSxLoss* a, hipStream_t s);
hipError_t jvk_sx_join(const float* part, int splits, int nq, const void* q, int64_t q_stride, const void* v, int64_t v_stride, int dtype, int d,
                       const int32_t* targets, int64_t n, float scale, float* loss, float* lse, hipStream_t s);
hipError_t jvk_sx_weights(const JvSxWeights* a, hipStream_t s);
hipError_t jvk_sx_mm(const JvMmOut* a, hipStream_t s);
hipError_t jvk_sx_finish(const float* slab, int splits, int64_t rows, int d, void* out, int dtype, int64_t ldo, hipStream_t s);
hipError_t jvk_sx_fill(void* out, int dtype, int64_t stride, int64_t rows, int d, float value, hipStream_t s);
}
