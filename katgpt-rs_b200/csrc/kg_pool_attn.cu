// kg_pool_attn.cu — kg_pool_attend_dev: attention of new rows over a paged K/V
// pool, ragged over requests.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kg_pdl.cuh"
#include "kg_serve.h"

namespace kg {
namespace serve {
namespace {

struct AttendArgs {
    kg_pool p;
    int n_req, n_head, group, total_q, width, causal;
    const int32_t *cu, *kv, *table;
    const void *q;
    void *out;
    int64_t q_row, q_head, o_row, o_head;
    float scale;
    int *err;
};

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }

// Whether request r's lengths can be used (reported otherwise).
__device__ __forceinline__ bool request_ok(const AttendArgs &a, int r) {
    const int q0 = a.cu[r], q1 = a.cu[r + 1], kv = a.kv[r];
    return q0 >= 0 && q1 >= q0 && q1 <= a.total_q && kv >= 0 && kv <= (int64_t)a.width * a.p.page_size;
}

// One warp per (row, query head): a running maximum and sum over the row's
// positions, one position at a time.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_rows_kernel(AttendArgs a) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int row = (int)(w / a.n_head), h = (int)(w % a.n_head);
    if (row >= a.total_q) return;
    int r = -1;
    for (int i = lane; i < a.n_req; i += 32)
        if (request_ok(a, i)) {
            if (row >= a.cu[i] && row < a.cu[i + 1]) r = i;
        } else {
            atomicExch(a.err, (int)KG_ERR_INVALID_ARG);
        }
    for (int d = 16; d; d >>= 1) r = max(r, __shfl_xor_sync(~0u, r, d));
    if (r < 0) return;
    const int kv = a.kv[r], at = kv - a.cu[r + 1] + row, n = a.causal ? min(at + 1, kv) : kv;
    constexpr int E = D / 32;
    const T *q = static_cast<const T *>(a.q) + row * a.q_row + h * a.q_head + lane * E;
    const int hk = h / a.group;
    float qf[E], o[E], m = -INFINITY, l = 0.0f;
    for (int e = 0; e < E; ++e) {
        qf[e] = to_f(q[e]) * a.scale;
        o[e] = 0.0f;
    }
    for (int j = 0; j < n; ++j) {
        const int page = a.table[(int64_t)r * a.width + j / a.p.page_size];
        const bool ok = page >= 0 && page < a.p.n_pages;
        if (!ok) atomicExch(a.err, (int)KG_ERR_INVALID_ARG);
        const int64_t off = ok ? page * a.p.page_stride + (j % a.p.page_size) * a.p.row_stride + hk * a.p.head_stride + lane * E : 0;
        float s = 0.0f;
        for (int e = 0; e < E; ++e) s += ok ? qf[e] * to_f(static_cast<const T *>(a.p.k)[off + e]) : 0.0f;
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
        const float mn = fmaxf(m, s), c = __expf(m - mn), p = __expf(s - mn);
        l = l * c + p;
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + (ok ? p * to_f(static_cast<const T *>(a.p.v)[off + e]) : 0.0f);
        m = mn;
    }
    T *out = static_cast<T *>(a.out) + row * a.o_row + h * a.o_head + lane * E;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    for (int e = 0; e < E; ++e) out[e] = from_f<T>(o[e] * inv);
}

template <typename T>
cudaError_t launch(const AttendArgs &a, cudaStream_t s) {
    const dim3 grid((unsigned)(((int64_t)a.total_q * a.n_head + 3) / 4));
    if (a.p.head_dim == 64) return launch_pdl(attend_rows_kernel<T, 64>, grid, dim3(128), 0, s, a);
    return launch_pdl(attend_rows_kernel<T, 128>, grid, dim3(128), 0, s, a);
}

int check(kg_ctx *ctx, const kg_pool *pool, int32_t n_req, int32_t n_head, int32_t total_q) {
    if (int rc = check_pool(ctx, pool)) return rc;
    if (n_req < 0 || total_q < 0) return fail(ctx, KG_ERR_INVALID_ARG, "attend: n_req and total_q must not be negative");
    if (n_req > kMaxReq) return fail(ctx, KG_ERR_UNSUPPORTED, "attend: at most 16384 requests");
    if (n_head < 1 || n_head % pool->n_kv_head)
        return fail(ctx, KG_ERR_INVALID_ARG, "attend: n_head must be a multiple of the pool's n_kv_head");
    if (n_head / pool->n_kv_head > 64) return fail(ctx, KG_ERR_UNSUPPORTED, "attend: at most 64 query heads a K/V head");
    if ((int64_t)total_q * n_head > INT32_MAX) return fail(ctx, KG_ERR_UNSUPPORTED, "attend: total_q * n_head must stay below 2^31");
    return KG_OK;
}

}  // namespace
}  // namespace serve
}  // namespace kg

extern "C" {

int64_t kg_pool_attend_bytes(const kg_pool *pool, int32_t n_req, int32_t n_head, int32_t total_q) {
    if (int rc = kg::serve::check(nullptr, pool, n_req, n_head, total_q)) return rc;
    return 16;
}

int kg_pool_attend_dev(kg_ctx *ctx, const kg_pool *pool, int32_t n_req, int32_t n_head, int32_t total_q,
                       const int32_t *cu_q, const int32_t *kv_len, const int32_t *table, int32_t table_width,
                       const void *q, int64_t q_row_stride, int64_t q_head_stride, void *out, int64_t out_row_stride,
                       int64_t out_head_stride, float scale, int32_t causal, void *workspace, int64_t workspace_bytes,
                       void *stream) {
    using namespace kg::serve;
    if (int rc = check(ctx, pool, n_req, n_head, total_q)) return rc;
    if (table_width < 1) return fail(ctx, KG_ERR_INVALID_ARG, "attend: table_width must be positive");
    const bool some = n_req > 0 && total_q > 0;
    if (some) {
        if (!cu_q || !kv_len || !table || !q || !out || !workspace) return fail(ctx, KG_ERR_INVALID_ARG, "attend: null pointer");
        if (q == out) return fail(ctx, KG_ERR_INVALID_ARG, "attend: q and out must not overlap");
        if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || q_row_stride % 8 || q_head_stride % 8 ||
            out_row_stride % 8 || out_head_stride % 8)
            return fail(ctx, KG_ERR_INVALID_ARG, "attend: bases must be 16-byte aligned and strides multiples of 8");
        if (q_row_stride < 0 || q_head_stride < 0 || out_row_stride < 0 || out_head_stride < 0 ||
            !nested(pool->head_dim, {q_row_stride, total_q}, {q_head_stride, n_head}, {0, 1}) ||
            !nested(pool->head_dim, {out_row_stride, total_q}, {out_head_stride, n_head}, {0, 1}))
            return fail(ctx, KG_ERR_INVALID_ARG, "attend: rows overlap at these strides");
        if (workspace_bytes < kg_pool_attend_bytes(pool, n_req, n_head, total_q))
            return fail(ctx, KG_ERR_INVALID_ARG, "attend: workspace smaller than kg_pool_attend_bytes");
        if (!(scale > -INFINITY && scale < INFINITY)) return fail(ctx, KG_ERR_INVALID_ARG, "attend: scale must be finite");
    }
    if (!ctx) return fail(ctx, KG_ERR_INVALID_ARG, "null context");
    if (!some) return KG_OK;
    DeviceGuard dg(ctx->device);
    if (dg.err != cudaSuccess) return cuda_fail(ctx, dg.err, "kg_pool_attend_dev");
    AttendArgs a{*pool, n_req, n_head, n_head / pool->n_kv_head, total_q, table_width, causal, cu_q, kv_len, table, q, out,
                 q_row_stride, q_head_stride, out_row_stride, out_head_stride, scale, ctx->serve_err};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = pool->dtype == KG_DT_BF16 ? launch<__nv_bfloat16>(a, s) : launch<__half>(a, s);
    return e == cudaSuccess ? KG_OK : cuda_fail(ctx, e, "kg_pool_attend_dev");
}

}  // extern "C"
