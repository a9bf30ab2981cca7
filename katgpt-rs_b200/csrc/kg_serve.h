// kg_serve.h — host side shared by the serving operators over a caller-owned
// page pool (kg_pool.cu, kg_pool_attn.cu, kg_logits.cu): argument checks,
// error messages with and without a context, and the caller's device.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "kg_internal.h"

namespace kg {
namespace serve {

constexpr int kMaxReq = 16384;     // requests of one call
constexpr int kMaxVocab = 262144;  // 2^18 weights of at most 2^44 sum below 2^63

#ifdef __CUDACC__
// An argument that a device-side check turned down, for kg_pool_status. KG_ERR_TIMEOUT, the lower number, stays: it is
// about every row of a call, not about the ones that were named.
__device__ __forceinline__ void reject(int *err) { atomicMin(err, (int)KG_ERR_INVALID_ARG); }
static_assert(KG_ERR_TIMEOUT < KG_ERR_INVALID_ARG && KG_ERR_INVALID_ARG < KG_OK, "the lowest status stays");
#endif

// Message of the calling thread's last call without a context.
std::string &thread_error();
inline int fail(kg_ctx *ctx, int code, const std::string &msg) {
    (ctx ? ctx->err : thread_error()) = msg;
    return code;
}
inline int cuda_fail(kg_ctx *ctx, cudaError_t e, const char *what) {
    return fail(ctx, e == cudaErrorMemoryAllocation ? KG_ERR_OOM : KG_ERR_CUDA,
                std::string(what) + ": " + cudaGetErrorString(e));
}

// The context's device for the duration of a call, the caller's afterwards.
struct DeviceGuard {
    int before = -1;
    cudaError_t err;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
        else if (err == cudaSuccess) before = -1;  // nothing to put back
    }
    ~DeviceGuard() {
        if (before >= 0) (void)cudaSetDevice(before);
    }
};

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// No two of the rows that (stride, count) pairs span overlap: every stride
// steps over all that the smaller ones span (`row` contiguous elements inside).
struct Axis {
    int64_t stride, count;
};
inline bool nested(int64_t row, Axis a, Axis b, Axis c) {
    Axis x[3] = {a, b, c};
    std::sort(x, x + 3, [](const Axis &p, const Axis &q) { return p.stride < q.stride; });
    int64_t span = row;
    for (const Axis &v : x) {
        if (v.count <= 1) continue;
        if (v.stride < span) return false;
        if (v.stride > (INT64_MAX / 4 - span) / v.count) return false;  // element offsets stay far inside 64 bits
        span += v.stride * (v.count - 1);
    }
    return true;
}

// The greatest step (elements) that reaches every page and head.
inline int64_t pool_unit(const kg_pool &p) {
    int64_t a = p.n_pages > 1 ? p.page_stride : 0, b = p.n_kv_head > 1 ? p.head_stride : 0;
    while (b) {
        const int64_t t = a % b;
        a = b;
        b = t;
    }
    return a ? a : p.head_dim;
}

inline int check_pool(kg_ctx *ctx, const kg_pool *p) {
    if (!p) return fail(ctx, KG_ERR_INVALID_ARG, "null pool");
    if (!p->k || !p->v || p->k == p->v) return fail(ctx, KG_ERR_INVALID_ARG, "pool: k and v must be two device pointers");
    if (p->dtype != KG_DT_BF16 && p->dtype != KG_DT_F16)
        return fail(ctx, KG_ERR_UNSUPPORTED, "pool: dtype must be KG_DT_BF16 or KG_DT_F16");
    if (p->head_dim != 64 && p->head_dim != 128) return fail(ctx, KG_ERR_UNSUPPORTED, "pool: head_dim must be 64 or 128");
    if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128)
        return fail(ctx, KG_ERR_UNSUPPORTED, "pool: page_size must be 16, 32, 64 or 128");
    if (p->n_pages < 1 || p->n_kv_head < 1) return fail(ctx, KG_ERR_INVALID_ARG, "pool: n_pages and n_kv_head must be positive");
    if ((int64_t)p->n_pages * p->page_size > INT32_MAX)
        return fail(ctx, KG_ERR_INVALID_ARG, "pool: n_pages * page_size must stay below 2^31");
    if (!aligned16(p->k) || !aligned16(p->v) || p->page_stride % 8 || p->row_stride % 8 || p->head_stride % 8)
        return fail(ctx, KG_ERR_INVALID_ARG, "pool: bases must be 16-byte aligned and strides multiples of 8");
    if (p->page_stride < 0 || p->row_stride < 0 || p->head_stride < 0 ||
        !nested(p->head_dim, {p->page_stride, p->n_pages}, {p->row_stride, p->page_size}, {p->head_stride, p->n_kv_head}))
        return fail(ctx, KG_ERR_INVALID_ARG, "pool: rows overlap at these strides");
    const int64_t span = (p->n_pages > 1 ? (p->n_pages - 1) * p->page_stride : 0) + (p->n_kv_head > 1 ? (p->n_kv_head - 1) * p->head_stride : 0);
    if (span / pool_unit(*p) >= INT32_MAX || p->row_stride >= (int64_t)1 << 35)
        return fail(ctx, KG_ERR_UNSUPPORTED, "pool: page and head strides with a larger common divisor are needed for this many pages");
    return KG_OK;
}

}  // namespace serve
}  // namespace kg
