// jv_ops.h — argument blocks of the training and 8-bit scoring kernels (jv_kernels_f8.hip, jv_kernels_sx.hip), shared with jv_abi_ops.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// One matrix product C[M][N].  An operand lies with k along its rows (lda / ldb bytes apart, M / N of them), or with k across them
// (ka / kb rows, of ca / cb bf16 columns; what lies behind the last row reads as the last row again, so the OTHER operand holds zeros there).
// 8-bit and bf16 operands: k is whole phases of 64 B a row (32 bf16, 64 e4m3; an even number, zeros behind the data), everything is 4-B aligned
// and columns come in eights.  float32 operands: jv_tile32.h, jv_tile3.h.
struct JvMm {
    const char *a, *b;
    int64_t lda, ldb;
    int32_t M, N;
    int32_t k;               // components (float32)
    int32_t kph;             // phases (bf16, e4m3)
    int64_t plane_a;         // float32 as bf16 planes: bytes from plane to plane
    int32_t ka, kb, ca, cb;  // operands with k across their rows
    int32_t end_b;           // bytes of k that a row of B has, 16 at least (bf16, k along its rows): the 16 B that would pass its end, and those behind,
                             // are read from 16 B before it instead, and A holds the 16 B that pass its end in that order, zeros for what was there already
    const char* tail_b;      // bf16, k across B's rows: 16 B that stand for the last 16 B of columns of B's last row, which may pass the matrix's end
    const uint8_t *sa, *sb;  // e4m3: scale bytes [M][kph / 2] / [N][kph / 2]
};

// a product written as it is, times mul * *norm
struct JvMmOut {
    JvMm mm;
    float mul;
    const float* norm;     // nullptr = 1
    int32_t dtype;         // JV_DTYPE_*
    void* out;             // [M][ldo]
    int64_t ldo;           // elements
    int32_t splits;        // partial sums over `splits` k ranges, float32 [splits][M][ldo] at `out`
    int32_t add;           // to what is there (float32)
    const int32_t* targets;   // rows of C are queries, those without a target among `n` rows become zeros (jvs_grads_tile_kernel's first product); nullptr = all have one
    int64_t n;
};
// the logits' forward pass: A = queries, B = vectors
struct JvSxLoss {
    JvMm mm;
    float c;               // scale * log2(e)
    int32_t path;          // JvSxPath
    int32_t splits;        // jvk_sx_loss_splits
    float2* part;          // [M][splits]: maximum and sum (log2 domain) over the rows but for the target
    int32_t first;         // 0: partials of an earlier piece of the rows are in `part` already, join them
    const int32_t* targets;  // nullptr = none
    int64_t row0;          // first row of this piece
    float* hit;            // [M] the target's product, written by the piece that has it
};
// what the gradient needs of a query
struct JvSxQuery {
    float lse2;            // base-2 logarithm
    float w;               // weight / norm, times 2^-(what lse2 lacks of its value); 0 = the query takes no part
    int32_t target;        // row, -1 = none
    float own;             // weight / norm, to be taken off p at the target; where the losses are known, g there: weight / norm * (exp(-loss) - 1)
};
// partial sums of a gradient, [splits][rows][lds], to be joined
struct JvSxFinish {
    const float* slab;
    int32_t splits;
    int64_t rows;
    void* out;             // [rows][ldo]
    int64_t ldo;
    const float* rest;     // per row, times the row's target: added; nullptr = none
    const JvSxQuery* query;
    const void* vectors;
    int64_t v_stride;
    const int32_t* targets;   // rows without a target among `n` become zeros; nullptr = all have one
    int64_t n;
};
// One piece of the gradient's weights G = w (p - [j = target]), zeros where a query has no target: bf16 [M][kv]; float32 as three
// planes [M][3][kv] (JV_SX_PLANES) or as it is [M][kv] (JV_SX_RAW).  Behind the last query: zeros, one row of them or up to a multiple of 64.
struct JvSxWeights {
    JvMm mm;               // A = queries, B = vectors of this piece
    float c;
    int64_t row0;          // first row of this piece
    const JvSxQuery* query;   // nullptr: from lse, loss, w (nullptr = 1) and targets as they are
    const float *lse, *loss, *w;   // loss: nullptr = not known
    const int32_t* targets;
    int64_t n;             // rows in all
    int32_t path;          // JvSxPath
    void* g;
    int32_t kv;            // N padded to 64
    float* rest;           // [M] bf16: what G's entry at the target lacks of its float32 value
    float* clean;          // JV_SX_RAW: the queries [M][d], those without a target as zeros, written beside; nullptr = none
};

// what has to be laid out before a product: up to three matrices (rows -> bf16 planes [rows][planes][kp]) and the queries' constants, one launch
struct JvSxPrepare {
    struct Matrix {
        const void* x;
        int64_t stride, rows;   // rows = 0: none
        void* out;
        int32_t kp;
        int32_t raw;            // float32 rows [rows][kp] as they are
        int32_t clean;          // rows without a target become zeros
        int32_t shift;          // bf16: the last components as JvMm.end_b wants them of A
    } m[3];
    int32_t dtype, d;
    const int32_t* targets;     // of the queries, for n rows
    int64_t n;
    // the gradient's queries (query == nullptr: none)
    const float *lse, *loss, *w;
    int32_t nq;
    JvSxQuery* query;
    float *norm, *rest;
    const void* last;       // bf16: the last row, whose last components (a multiple of 8 of them in front) become `tail`; nullptr = none
    void* tail;
};

// sets jv_last_error() and returns `code` (jv_abi.cpp)
__attribute__((visibility("hidden"))) int jvi_fail(int code, const char* fmt, ...);

extern "C" {
hipError_t jvk_f8_encode(const void* x, int dtype, int64_t stride, int64_t n, int d, uint8_t* codes, uint8_t* scales, hipStream_t s);
hipError_t jvk_f8_decode(const uint8_t* codes, const uint8_t* scales, int64_t n, int d, void* x, int dtype, int64_t stride, hipStream_t s);
hipError_t jvk_f8_score(const JvMmOut* a, hipStream_t s);

hipError_t jvk_sx_prepare(const JvSxPrepare* a, hipStream_t s);
// How the products of a shape are computed.
enum JvSxPath {
    JV_SX_LARGE,    // bf16, 256 x 256 tiles (jv_pipe.h)
    JV_SX_TILES,    // bf16 on smaller tiles (jv_mm.h)
    JV_SX_PLANES,   // float32: queries and g as planes, vectors as they lie (jv_tile3.h)
    JV_SX_RAW       // float32, few tiles: everything as it lies (jv_tile32.h)
};
int jvk_sx_path(int nq, int64_t rows, int f32);
int jvk_sx_loss_splits(int path, int nq, int64_t rows, int d);   // workgroups that share a panel of queries
hipError_t jvk_sx_loss(const JvSxLoss* a, hipStream_t s);
hipError_t jvk_sx_join(const float2* part, int splits, int nq, float c, const float* hit, const int32_t* targets, int64_t n, float* loss, float* lse, hipStream_t s);
hipError_t jvk_sx_weights(const JvSxWeights* a, hipStream_t s);
// dq = G V and dv = G^T Q (nullptr: not asked for)
int jvk_sx_grad_splits(int path, int64_t rows, int d, int64_t k, int across);
hipError_t jvk_sx_grads(const JvMmOut* q, const JvMmOut* v, int path, hipStream_t s);
hipError_t jvk_sx_finish(const JvSxFinish* q, const JvSxFinish* v, int d, int64_t lds, float mul, const float* norm, int dtype, hipStream_t s);
hipError_t jvk_sx_fill(void* out, int dtype, int64_t stride, int64_t rows, int d, float value, hipStream_t s);
}
