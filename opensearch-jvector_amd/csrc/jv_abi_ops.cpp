// jv_abi_ops.cpp — C ABI of the training and 8-bit scoring operators (include/jvgpu.h): argument checks, plans, launches.
// No handle, no allocation, no host round trip: a call only enqueues kernels on the caller's stream, so it can be captured.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/jvgpu.h"
#include "jv_ops.h"

#define CHK(expr)                                                                                                                    \
    do {                                                                                                                             \
        hipError_t e_ = (expr);                                                                                                      \
        if (e_ != hipSuccess)                                                                                                        \
            return jvi_fail(e_ == hipErrorOutOfMemory ? JV_ENOMEM : JV_EDEVICE, "%s failed: %s", #expr, hipGetErrorString(e_));      \
    } while (0)

namespace {

constexpr int64_t kMaxRows = 0x7fffffffll - 65536;   // a tile behind the last row still has an int32 number
constexpr int64_t kMaxStride = 1ll << 31;
constexpr float kLog2E = 1.44269504088896341f;
constexpr int32_t kNoEnd = 0x7fffff00;          // JvMm.end_b of rows that have all of k

// the caller's current device comes back on every way out
class OnDevice {
public:
    explicit OnDevice(int device) {
        if ((err_ = hipGetDevice(&before_)) != hipSuccess) return;
        if (before_ != device && (err_ = hipSetDevice(device)) == hipSuccess) moved_ = true;
    }
    ~OnDevice() {
        if (moved_) (void)hipSetDevice(before_);
    }
    hipError_t error() const { return err_; }

private:
    int before_ = 0;
    bool moved_ = false;
    hipError_t err_ = hipSuccess;
};

int done(void* stream) {   // NULL: the legacy default stream, synchronous
    if (!stream) CHK(hipStreamSynchronize(nullptr));
    return JV_OK;
}

int size_of(int dtype) { return dtype == JV_DTYPE_F32 ? 4 : 2; }

int check_dtype(int dtype, const char* what) {
    if (dtype != JV_DTYPE_F32 && dtype != JV_DTYPE_BF16) return jvi_fail(JV_EINVAL, "%s: dtype %d is neither JV_DTYPE_F32 nor JV_DTYPE_BF16", what, dtype);
    return JV_OK;
}
// a matrix of the caller's: rows of d components, `stride` components apart
int check_rows(const void* p, int64_t rows, int64_t stride, int d, int dtype, const char* what) {
    if (rows > 0 && !p) return jvi_fail(JV_EINVAL, "%s is NULL", what);
    if ((uintptr_t)p % size_of(dtype)) return jvi_fail(JV_EINVAL, "%s is not aligned to its %d-byte components", what, size_of(dtype));
    if (stride < d || stride > kMaxStride) return jvi_fail(JV_EINVAL, "%s: row stride %lld not in [d = %d, 2^31]", what, (long long)stride, d);
    return JV_OK;
}
int check_codes(const void* codes, const void* scales, int64_t rows, const char* what) {
    if (rows > 0 && (!codes || !scales)) return jvi_fail(JV_EINVAL, "%s: codes / scales are NULL", what);
    if ((uintptr_t)codes % 16) return jvi_fail(JV_EINVAL, "%s: codes are not 16-byte aligned", what);
    return JV_OK;
}
int check_shape(int64_t n, int d, const char* what) {
    if (n < 0 || d <= 0) return jvi_fail(JV_EINVAL, "%s: bad shape n=%lld d=%d", what, (long long)n, d);
    if (n > kMaxRows || d > JV_OPS_MAX_D) return jvi_fail(JV_EUNSUPPORTED, "%s: n=%lld d=%d beyond %lld rows / %d components", what, (long long)n, d, (long long)kMaxRows, JV_OPS_MAX_D);
    return JV_OK;
}

#define TRY(x)                        \
    do {                              \
        const int rc_ = (x);          \
        if (rc_ != JV_OK) return rc_; \
    } while (0)

// ---- the softmax loss: what a call needs, from its shape alone ----
struct Plan {
    int P, dp, kq, gq;                // planes; d and nq padded to 64; rows of g (the large tiles write whole steps, the small ones one row behind the queries)
    int64_t rows_f, rows_b;           // rows of one piece, forward (where the vectors have to be laid out) / backward
    int path_f, path_b, splits_f, splits_q, splits_v;   // forward, backward
    int64_t off_q, off_clean, off_v, off_part, off_hit, off_query, off_norm, off_tail, off_rest, off_g, off_slab, off_slab_v, bytes;
};

// MB of one piece's weights g: few large pieces, for every piece writes and reads dq's partial sums again and starts its tiles anew (step
// 4096 x 131072 x 1024: 4.67 ms with 128, 4.54 with 384, 4.32 with 1024, all of it in one piece).  A piece has whole tiles of 256 rows and at least one: 6 GiB
// of g with 2^22 float32 queries.
constexpr int64_t kWeights = 1024;
// MB of one piece's rows, where a gradient needs them laid out
constexpr int64_t kLaid = 2048;

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// n cut into equal pieces of at most `most` rows, whole tiles
int64_t piece(int64_t n, int64_t most) {
    most = std::max<int64_t>(up(most, 256), 256);
    const int64_t pieces = std::max<int64_t>((n + most - 1) / most, 1);
    return std::max<int64_t>(up((n + pieces - 1) / pieces, 256), 256);
}

// The products take the vectors as they lie (take_rows): float32 with at least four components; bf16, 4-B aligned, with an even number of them,
// eight at least.
bool can_lie(int dtype, int d) { return dtype == JV_DTYPE_F32 ? d >= 4 : d >= 8 && d % 2 == 0; }
bool lies(const jv_softmax_params* p) {
    return can_lie(p->dtype, p->d) && (p->dtype == JV_DTYPE_F32 || ((uintptr_t)p->vectors % 4 == 0 && p->vector_stride % 2 == 0));
}

// `as_is`: the vectors are taken as they lie
Plan make_plan(int dtype, int nq, int64_t n, int d, uint32_t what, bool as_is) {
    Plan p{};
    p.P = dtype == JV_DTYPE_F32 ? 3 : 1;
    p.dp = (int)up(d, 64);
    p.kq = (int)up(std::max(nq, 1), 64);
    p.gq = nq > 128 ? p.kq : nq + 1;
    const int64_t panels = std::max((nq + 255) / 256, 1), row = (int64_t)p.P * p.dp * 2;
    const int64_t fill = 256 * ((1024 + panels - 1) / panels);   // rows whose tiles fill the chip four times
    p.rows_f = piece(n, std::max<int64_t>((128ll << 20) / row, fill));
    const int64_t most = (kWeights << 20) / ((int64_t)p.P * 2 * p.gq);
    p.rows_b = piece(n, std::max<int64_t>(as_is ? most : std::min(most, (kLaid << 20) / row), fill));
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += up(bytes, 256);
        return o;
    };
    // bytes of a query or row that is laid out: float32 of fewer than four components as four of them (rows_of), queries of JV_SX_RAW not at all otherwise
    const bool f32 = dtype == JV_DTYPE_F32;
    auto query = [&](int path) { return f32 && path == JV_SX_RAW ? d < 4 ? 16 : 0 : row; };
    const int64_t laid = f32 ? 16 : row;
    if (what & JV_SOFTMAX_LOSS) {
        p.path_f = jvk_sx_path(nq, n, f32);
        p.off_q = take(nq * query(p.path_f));
        p.splits_f = jvk_sx_loss_splits(p.path_f, nq, n, d);
        p.off_part = take((int64_t)p.splits_f * nq * 8);
        p.off_hit = take((int64_t)nq * 4);
        p.off_v = take(as_is ? 0 : std::min<int64_t>(p.rows_f, n) * laid);
    }
    if (what & (JV_SOFTMAX_QUERY_GRAD | JV_SOFTMAX_VECTOR_GRAD)) {
        p.path_b = jvk_sx_path(nq, std::min<int64_t>(p.rows_b, n), f32);
        p.off_q = take(nq * query(p.path_b));
        p.off_v = take(as_is ? 0 : std::min<int64_t>(p.rows_b, n) * laid);
        p.off_query = take((int64_t)nq * sizeof(JvSxQuery));
        p.off_norm = take(4);
        p.off_tail = take(16);
        p.off_rest = take((int64_t)nq * 4);
        p.off_g = take((int64_t)p.gq * p.P * p.rows_b * 2);
        if (what & JV_SOFTMAX_QUERY_GRAD) {
            p.splits_q = jvk_sx_grad_splits(p.path_b, nq, d, std::min<int64_t>(p.rows_b, n), 0);
            p.off_slab = take((int64_t)p.splits_q * nq * p.dp * 4);
        }
        if (what & JV_SOFTMAX_VECTOR_GRAD) {
            const int64_t rows = std::min<int64_t>(p.rows_b, n);
            p.splits_v = jvk_sx_grad_splits(p.path_b, rows, d, nq, 1);
            p.off_clean = take(f32 ? (int64_t)nq * std::max(d, 4) * 4 : d % 8 ? (int64_t)nq * p.dp * 2 : 0);
            p.off_slab_v = take(p.splits_v > 1 ? p.splits_v * rows * p.dp * 4 : 0);
        }
    }
    p.bytes = at;
    return p;
}

// Rows as a product takes them: the caller's own (the vectors where lies(); queries in bf16 where they are 4-B aligned and whole steps of 64, for
// their padding stands for zeros behind the vectors', and in float32 where the path takes them as they lie), or laid out.
struct Rows {
    const char* p;
    int64_t stride;   // bytes
    bool ready;
    int kp;           // components of a row that is laid out instead
    bool raw;         // as float32, not as planes
    int cols(int d) const { return raw ? d : ready ? (int)up(d, 8) : kp; }
};
Rows rows_of(const void* p, int64_t stride, const jv_softmax_params* q, const Plan& plan, int path, bool vectors) {
    Rows r{(const char*)p, stride * size_of(q->dtype), false, plan.dp, false};
    if (q->dtype == JV_DTYPE_BF16) r.ready = vectors ? lies(q) : (uintptr_t)p % 4 == 0 && stride % 2 == 0 && q->d % 64 == 0;
    else if (path == JV_SX_RAW || vectors) r.ready = q->d >= 4, r.kp = 4, r.raw = true;
    return r;
}

int check_softmax(const jv_softmax_params* p) {
    if (!p) return jvi_fail(JV_EINVAL, "softmax: params is NULL");
    if (p->struct_size != sizeof(jv_softmax_params))
        return jvi_fail(JV_EINVAL, "jv_softmax_params.struct_size %u != %zu (ABI mismatch)", p->struct_size, sizeof(jv_softmax_params));
    TRY(check_dtype(p->dtype, "softmax"));
    TRY(check_shape(p->n, p->d, "softmax: vectors"));
    TRY(check_shape(p->nq, p->d, "softmax: queries"));
    if (p->nq > JV_SOFTMAX_MAX_QUERIES) return jvi_fail(JV_EUNSUPPORTED, "softmax: %d queries (> %d)", p->nq, JV_SOFTMAX_MAX_QUERIES);
    if (!std::isfinite(p->scale * kLog2E)) return jvi_fail(JV_EINVAL, "softmax: scale or its product with log2(e) is not finite");
    return JV_OK;
}
int check_softmax_call(const jv_softmax_params* p, const Plan& plan) {
    TRY(check_rows(p->queries, p->nq, p->query_stride, p->d, p->dtype, "softmax: queries"));
    TRY(check_rows(p->vectors, p->n, p->vector_stride, p->d, p->dtype, "softmax: vectors"));
    if (!p->workspace || (uintptr_t)p->workspace % 256) return jvi_fail(JV_EINVAL, "softmax: workspace is NULL or not 256-byte aligned");
    if (p->workspace_bytes < plan.bytes)
        return jvi_fail(JV_EINVAL, "softmax: workspace of %lld bytes, %lld needed", (long long)p->workspace_bytes, (long long)plan.bytes);
    return JV_OK;
}

// k ranges that a piece of `rows` rows has at most: its steps
int splits_of(const Plan& plan, int64_t rows) {
    return (int)(up(rows, 64) / (plan.path_b == JV_SX_RAW || plan.path_b == JV_SX_PLANES ? 32 : 64));
}

// queries times vectors, but for where the vectors lie and how many they are
JvMm logits(const Plan& plan, int nq, int d) {
    JvMm mm{};
    mm.M = nq, mm.k = d, mm.kph = plan.dp / 32;
    mm.plane_a = (int64_t)plan.dp * 2;
    mm.end_b = kNoEnd;
    return mm;
}

// The rows [at, at + rows) of a matrix as a product reads them: the caller's own, or where the next jvk_sx_prepare lays them out.
void take_rows(const Rows& r, int dtype, int64_t at, int64_t rows, const Plan& plan, char* to, JvSxPrepare::Matrix* m, const char** out, int64_t* ld) {
    if (r.ready) {
        *out = r.p + at * r.stride;
        *ld = r.stride;
        m->rows = 0;
        return;
    }
    m->x = r.p + at * r.stride, m->stride = r.stride / size_of(dtype), m->rows = rows, m->out = to, m->kp = r.kp, m->raw = r.raw;
    *out = to;
    *ld = r.raw ? (int64_t)r.kp * 4 : (int64_t)plan.P * plan.dp * 2;
}

}  // namespace

extern "C" {

int jv_encode_blocks_device(int32_t device, const void* d_vectors, int32_t dtype, int64_t row_stride, int32_t n, int32_t d, uint8_t* d_out_codes,
                            uint8_t* d_out_scales, void* hip_stream) {
    TRY(check_dtype(dtype, "encode"));
    TRY(check_shape(n, d, "encode"));
    TRY(check_rows(d_vectors, n, row_stride, d, dtype, "encode: vectors"));
    TRY(check_codes(d_out_codes, d_out_scales, n, "encode"));
    OnDevice on(device);
    CHK(on.error());
    CHK(jvk_f8_encode(d_vectors, dtype, row_stride, n, d, d_out_codes, d_out_scales, (hipStream_t)hip_stream));
    return done(hip_stream);
}

int jv_decode_blocks_device(int32_t device, const uint8_t* d_codes, const uint8_t* d_scales, int32_t n, int32_t d, int32_t dtype, void* d_out_vectors,
                            int64_t row_stride, void* hip_stream) {
    TRY(check_dtype(dtype, "decode"));
    TRY(check_shape(n, d, "decode"));
    TRY(check_rows(d_out_vectors, n, row_stride, d, dtype, "decode: vectors"));
    TRY(check_codes(d_codes, d_scales, n, "decode"));
    OnDevice on(device);
    CHK(on.error());
    CHK(jvk_f8_decode(d_codes, d_scales, n, d, d_out_vectors, dtype, row_stride, (hipStream_t)hip_stream));
    return done(hip_stream);
}

int jv_score_blocks_device(int32_t device, const uint8_t* d_query_codes, const uint8_t* d_query_scales, int32_t nq, const uint8_t* d_codes,
                           const uint8_t* d_scales, int32_t n, int32_t d, int32_t dtype, void* d_out_scores, int64_t row_stride, void* hip_stream) {
    TRY(check_dtype(dtype, "score"));
    TRY(check_shape(nq, d, "score: queries"));
    TRY(check_shape(n, d, "score: rows"));
    TRY(check_codes(d_query_codes, d_query_scales, nq, "score: queries"));
    TRY(check_codes(d_codes, d_scales, n, "score: rows"));
    if (nq > 0) TRY(check_rows(d_out_scores, n, row_stride, n, dtype, "score: scores"));
    OnDevice on(device);
    CHK(on.error());
    JvMmOut a{};
    const int blocks = (d + 127) / 128;
    a.mm.kph = 2 * blocks;
    a.mm.a = (const char*)d_query_codes, a.mm.b = (const char*)d_codes;
    a.mm.lda = a.mm.ldb = (int64_t)blocks * 128;
    a.mm.M = nq, a.mm.N = n, a.mm.end_b = kNoEnd;
    a.mm.sa = d_query_scales, a.mm.sb = d_scales;
    a.mul = 1.0f, a.dtype = dtype, a.out = d_out_scores, a.ldo = row_stride, a.splits = 1;
    CHK(jvk_f8_score(&a, (hipStream_t)hip_stream));
    return done(hip_stream);
}

int jv_softmax_workspace(const jv_softmax_params* params, uint32_t what, int64_t* out_bytes) {
    TRY(check_softmax(params));
    if (!out_bytes || !(what & 7u) || (what & ~15u)) return jvi_fail(JV_EINVAL, "softmax: out_bytes is NULL, no call is named or unknown flags %#x", what);
    const bool here = what & JV_SOFTMAX_AS_THEY_LIE;
    int64_t need = 256;   // (the loss and its gradient are separate calls: the larger of the two)
    for (uint32_t part : {what & JV_SOFTMAX_LOSS, what & (JV_SOFTMAX_QUERY_GRAD | JV_SOFTMAX_VECTOR_GRAD)})
        for (bool as_is : {false, true})   // (bf16: where the vectors lie decides)
            if (part && (here ? as_is == lies(params) : as_is ? can_lie(params->dtype, params->d) : params->dtype == JV_DTYPE_BF16 || !can_lie(params->dtype, params->d)))
                need = std::max(need, make_plan(params->dtype, params->nq, params->n, params->d, part, as_is).bytes);
    *out_bytes = need;
    return JV_OK;
}

int jv_softmax_loss_device(const jv_softmax_params* p, float* d_out_loss, float* d_out_lse, void* hip_stream) {
    TRY(check_softmax(p));
    const Plan plan = make_plan(p->dtype, p->nq, p->n, p->d, JV_SOFTMAX_LOSS, lies(p));
    TRY(check_softmax_call(p, plan));
    if (p->nq > 0 && (!d_out_loss || !d_out_lse)) return jvi_fail(JV_EINVAL, "softmax: output pointer is NULL");
    OnDevice on(p->device);
    CHK(on.error());
    hipStream_t s = (hipStream_t)hip_stream;
    if (p->nq > 0) {
        char* ws = (char*)p->workspace;
        const Rows rq = rows_of(p->queries, p->query_stride, p, plan, plan.path_f, false), rv = rows_of(p->vectors, p->vector_stride, p, plan, plan.path_f, true);
        const int64_t step = rv.ready ? std::max<int64_t>(p->n, 1) : plan.rows_f;
        JvSxLoss a{};
        a.mm = logits(plan, p->nq, p->d);
        a.c = p->scale * kLog2E;
        a.targets = p->targets, a.hit = (float*)(ws + plan.off_hit);
        const bool shift = rv.ready && p->dtype == JV_DTYPE_BF16 && p->d % 8;   // (JvMm.end_b)
        if (rv.ready && p->dtype == JV_DTYPE_BF16) a.mm.end_b = p->d * 2;
        a.path = plan.path_f, a.splits = p->n > 0 ? plan.splits_f : 0, a.part = (float2*)(ws + plan.off_part);
        JvSxPrepare pre{};
        pre.dtype = p->dtype, pre.d = p->d;
        take_rows(rq, p->dtype, 0, p->nq, plan, ws + plan.off_q, &pre.m[0], &a.mm.a, &a.mm.lda);
        pre.m[0].shift = shift;
        for (int64_t at = 0; at < p->n; at += step) {
            a.mm.N = (int)std::min<int64_t>(step, p->n - at);
            a.first = at == 0, a.row0 = at;
            take_rows(rv, p->dtype, at, a.mm.N, plan, ws + plan.off_v, &pre.m[1], &a.mm.b, &a.mm.ldb);
            CHK(jvk_sx_prepare(&pre, s));
            pre.m[0].rows = 0;
            CHK(jvk_sx_loss(&a, s));
        }
        CHK(jvk_sx_join(a.part, a.splits, p->nq, a.c, a.hit, p->targets, p->n, d_out_loss, d_out_lse, s));
    }
    return done(hip_stream);
}

int jv_softmax_grad_device(const jv_softmax_params* p, const float* d_lse, const float* d_loss_grad, void* d_out_query_grad, int64_t query_grad_stride,
                           void* d_out_vector_grad, int64_t vector_grad_stride, void* hip_stream) {
    return jv_softmax_grad_device_ex(p, d_lse, nullptr, d_loss_grad, d_out_query_grad, query_grad_stride, d_out_vector_grad, vector_grad_stride, hip_stream);
}

int jv_softmax_grad_device_ex(const jv_softmax_params* p, const float* d_lse, const float* d_loss, const float* d_loss_grad, void* d_out_query_grad,
                              int64_t query_grad_stride, void* d_out_vector_grad, int64_t vector_grad_stride, void* hip_stream) {
    TRY(check_softmax(p));
    const uint32_t what = (d_out_query_grad ? JV_SOFTMAX_QUERY_GRAD : 0) | (d_out_vector_grad ? JV_SOFTMAX_VECTOR_GRAD : 0);
    if (!what) return jvi_fail(JV_EINVAL, "softmax: no gradient asked for");
    const Plan plan = make_plan(p->dtype, p->nq, p->n, p->d, what, lies(p));
    TRY(check_softmax_call(p, plan));
    if (p->nq > 0 && !d_lse) return jvi_fail(JV_EINVAL, "softmax: lse is NULL");
    if (d_out_query_grad) TRY(check_rows(d_out_query_grad, p->nq, query_grad_stride, p->d, p->dtype, "softmax: query gradient"));
    if (d_out_vector_grad) TRY(check_rows(d_out_vector_grad, p->n, vector_grad_stride, p->d, p->dtype, "softmax: vector gradient"));
    OnDevice on(p->device);
    CHK(on.error());
    hipStream_t s = (hipStream_t)hip_stream;
    if (p->nq == 0 || p->n == 0 || !p->targets) {   // nothing was asked of the rows: gradients of zero
        if (d_out_query_grad) CHK(jvk_sx_fill(d_out_query_grad, p->dtype, query_grad_stride, p->nq, p->d, 0.0f, s));
        if (d_out_vector_grad) CHK(jvk_sx_fill(d_out_vector_grad, p->dtype, vector_grad_stride, p->n, p->d, 0.0f, s));
        return done(hip_stream);
    }
    char* ws = (char*)p->workspace;
    Rows rq = rows_of(p->queries, p->query_stride, p, plan, plan.path_b, false);
    const Rows rv = rows_of(p->vectors, p->vector_stride, p, plan, plan.path_b, true);
    const bool f32 = p->dtype == JV_DTYPE_F32, raw = plan.path_b == JV_SX_RAW;
    JvSxWeights w{};
    w.mm = logits(plan, p->nq, p->d);
    w.c = p->scale * kLog2E;
    if (rv.ready && !f32) w.mm.end_b = p->d * 2;
    w.path = plan.path_b, w.g = ws + plan.off_g, w.loss = d_loss;
    // float32 g needs no common unit and lacks nothing at a target
    JvSxPrepare pre{};
    pre.dtype = p->dtype, pre.d = p->d;
    float* norm = nullptr;
    JvSxQuery* query = nullptr;
    if (f32) {
        w.lse = d_lse, w.w = d_loss_grad, w.targets = p->targets, w.n = p->n;
    } else {
        w.query = query = (JvSxQuery*)(ws + plan.off_query), w.rest = (float*)(ws + plan.off_rest), norm = (float*)(ws + plan.off_norm);
        pre.lse = d_lse, pre.loss = d_loss, pre.w = d_loss_grad, pre.nq = p->nq, pre.query = query, pre.norm = norm, pre.rest = w.rest;
    }
    const bool direct = raw && plan.splits_q == 1 && plan.rows_b >= p->n;   // dq is complete at once
    // Queries without a target are laid out as zeros.  dv's product reads them so: bf16 as they are laid out (again if the end is shifted),
    // float32 as a copy.
    const char* q_rows = ws + plan.off_clean;
    int64_t q_ld = (int64_t)p->d * 4;
    pre.targets = p->targets, pre.n = p->n;
    if (!f32) rq.ready = false;
    Rows rb = rq;
    take_rows(rq, p->dtype, 0, p->nq, plan, ws + plan.off_q, &pre.m[0], &w.mm.a, &w.mm.lda);
    pre.m[0].clean = !rq.ready;
    const bool shift = rv.ready && !f32 && p->d % 8;   // (JvMm.end_b)
    if (shift) {
        pre.m[0].shift = 1;
        if (d_out_query_grad) pre.last = (const char*)p->vectors + (int64_t)(p->n - 1) * p->vector_stride * 2, pre.tail = ws + plan.off_tail;
    }
    if (shift && d_out_vector_grad) {
        take_rows(rq, p->dtype, 0, p->nq, plan, ws + plan.off_clean, &pre.m[2], &q_rows, &q_ld);
        pre.m[2].clean = 1;
    } else if (!rq.ready && (!f32 || rq.raw)) {
        q_rows = w.mm.a, q_ld = w.mm.lda;
    } else if (d_out_vector_grad && plan.path_b == JV_SX_PLANES) {
        rb = rows_of(p->queries, p->query_stride, p, plan, JV_SX_RAW, false);
        rb.ready = false, rb.kp = std::max(p->d, 4);
        take_rows(rb, p->dtype, 0, p->nq, plan, ws + plan.off_clean, &pre.m[2], &q_rows, &q_ld);
        pre.m[2].clean = 1;
    } else if (d_out_vector_grad) {
        w.clean = (float*)(ws + plan.off_clean);
    }
    JvSxFinish fq{}, fv{};
    if (d_out_query_grad) {
        fq.slab = (const float*)(ws + plan.off_slab), fq.splits = std::min(plan.splits_q, splits_of(plan, std::min<int64_t>(plan.rows_b, p->n)));
        fq.rows = p->nq, fq.out = d_out_query_grad, fq.ldo = query_grad_stride;
        fq.rest = w.rest, fq.query = query, fq.vectors = p->vectors, fq.v_stride = p->vector_stride;
        fq.targets = p->targets, fq.n = p->n;
    }
    for (int64_t at = 0; at < p->n; at += plan.rows_b) {
        const int rows = (int)std::min<int64_t>(plan.rows_b, p->n - at);
        w.mm.N = rows, w.row0 = at, w.kv = (int)up(rows, 64);
        take_rows(rv, p->dtype, at, rows, plan, ws + plan.off_v, &pre.m[1], &w.mm.b, &w.mm.ldb);
        CHK(jvk_sx_prepare(&pre, s));
        pre.m[0].rows = pre.m[2].rows = 0, pre.query = nullptr;
        CHK(jvk_sx_weights(&w, s));
        JvMmOut o{}, q;
        o.mm.a = (const char*)w.g, o.mm.lda = raw ? (int64_t)w.kv * 4 : (int64_t)plan.P * w.kv * 2, o.mm.plane_a = (int64_t)w.kv * 2;
        o.mm.N = p->d, o.mm.end_b = kNoEnd;
        if (d_out_query_grad) {   // G times the piece's vectors: k = its rows
            o.mm.M = p->nq, o.mm.k = w.kv, o.mm.kph = w.kv / 32;
            o.mm.b = w.mm.b, o.mm.ldb = w.mm.ldb, o.mm.kb = rows, o.mm.cb = rv.cols(p->d);
            o.mm.tail_b = shift && at + rows == p->n ? ws + plan.off_tail : nullptr;
            o.mul = 1.0f, o.out = ws + plan.off_slab, o.ldo = plan.dp, o.add = at > 0;
            o.splits = std::min(plan.splits_q, splits_of(plan, rows));   // (only the last piece can be that short: it adds to the first ranges)
            if (direct) o.mul = p->scale, o.out = d_out_query_grad, o.ldo = query_grad_stride;
            q = o;
            if (direct) q.targets = p->targets, q.n = p->n;
            o.mm.tail_b = nullptr;
        }
        if (d_out_vector_grad) {   // G across times the queries: k = the queries
            o.mm.M = rows, o.mm.k = (int)up(p->nq, 32), o.mm.kph = plan.kq / 32, o.mm.ka = p->nq % (f32 ? 32 : 64) ? p->nq + 1 : p->nq, o.mm.ca = w.kv;
            o.mm.b = q_rows, o.mm.ldb = q_ld, o.mm.kb = p->nq, o.mm.cb = rb.cols(p->d);
            o.splits = plan.splits_v, o.add = 0;
            fv.out = (char*)d_out_vector_grad + at * vector_grad_stride * size_of(p->dtype), fv.ldo = vector_grad_stride;
            if (plan.splits_v > 1) {
                o.mul = 1.0f, o.out = ws + plan.off_slab_v, o.ldo = plan.dp;
                fv.slab = (const float*)o.out, fv.splits = o.splits, fv.rows = rows;
            } else {
                o.mul = p->scale, o.norm = norm, o.dtype = p->dtype, o.out = fv.out, o.ldo = fv.ldo;
            }
        }
        CHK(jvk_sx_grads(d_out_query_grad ? &q : nullptr, d_out_vector_grad ? &o : nullptr, plan.path_b, s));
        const bool join_q = d_out_query_grad && !direct && at + plan.rows_b >= p->n, join_v = fv.slab;
        if (join_q || join_v) CHK(jvk_sx_finish(join_q ? &fq : nullptr, join_v ? &fv : nullptr, p->d, plan.dp, p->scale, norm, p->dtype, s));
    }
    return done(hip_stream);
}

}  // extern "C"
