// kg_pool.cu — plan and store of the serving operators over a caller-owned
// page pool: block tables and slot maps from request lengths, and new K/V rows
// into their pages.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kg_dev.cuh"
#include "kg_pdl.cuh"
#include "kg_serve.h"

namespace kg {
namespace serve {

std::string &thread_error() {
    static thread_local std::string msg = "null context";
    return msg;
}

namespace {

// ---------------------------------------------------------------------------
// Plan. With c cached and n new positions and pages of P, request r holds
// has = ceil(c / P) pages and needs ceil((c + n) / P); two running sums over
// the requests (new tokens, new pages) place everything: page i of the step is
// free[n_free - 1 - i] and belongs to the request whose page range holds i,
// token t to the request whose token range holds t.
// Bound by latency: one launch. A cluster of 1 or 8 CTAs; each computes the running
// sums for itself (a few loads a thread), the checks meet at a cluster barrier
// before anything is written, and the tokens and pages are shared out. 512 ragged
// requests of 64 K tokens: 77 us by one CTA, 12.6 us a call by eight; 64 single tokens:
// 3.7 us in a graph, 9.8 us a call, the host's time.
struct PlanArgs {
    int page, n_pages, n_req, width, max_tokens;
    const int32_t *cached, *fresh;
    int32_t *table;
    const int32_t *free_pages, *n_free;
    int32_t *n_free_out, *cu, *kv, *slots, *req, *pos, *status;
};

constexpr int PLAN_THREADS = 1024;

// index of the range of the running sum `cum` (n + 1 entries) that holds i
__device__ __forceinline__ int range_of(const int32_t *cum, int n, int i) {
    int lo = 0, hi = n - 1;  // the answer: the last r with cum[r] <= i
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cum[mid] <= i) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
__device__ __forceinline__ int pages_of(long long positions, int shift) { return (int)((positions + (1 << shift) - 1) >> shift); }

__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(PlanArgs a) {
    extern __shared__ int32_t sm[];
    int32_t *cu = sm, *pg = sm + a.n_req + 1, *old = pg + a.n_req + 1;  // running sums of new tokens and new pages; cached lengths
    __shared__ long long wt[32], wp[32], s_tot[2];
    __shared__ int s_bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t rank, ctas;
    asm("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %cluster_nctarank;" : "=r"(ctas));
    const int shift = 31 - __clz(a.page), gid = (int)rank * PLAN_THREADS + tid, step = (int)ctas * PLAN_THREADS;
    if (tid == 0) s_bad = 0;
    pdl_wait();
    const int nf = *a.n_free;
    const int per = (a.n_req + PLAN_THREADS - 1) / PLAN_THREADS;
    const int r0 = min(tid * per, a.n_req), r1 = min(r0 + per, a.n_req);
    long long t = 0, p = 0;
    bool bad = nf < 0 || nf > a.n_pages;
    for (int r = r0; r < r1; ++r) {
        const long long c = a.cached[r], n = a.fresh[r], end = c + n;
        if (c < 0 || n < 0 || end > INT32_MAX || pages_of(end, shift) > a.width) {
            bad = true;
            continue;
        }
        old[r] = (int)c;
        if (n > 0 && c & (a.page - 1)) {  // its last page takes new rows
            const int e = a.table[(int64_t)r * a.width + (c >> shift)];
            bad |= e < 0 || e >= a.n_pages;
        }
        t += n;
        p += pages_of(end, shift) - pages_of(c, shift);
    }
    long long it = t, ip = p;  // inclusive sums over the block's threads
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long u = __shfl_up_sync(~0u, it, d), v = __shfl_up_sync(~0u, ip, d);
        if (lane >= d) {
            it += u;
            ip += v;
        }
    }
    if (lane == 31) {
        wt[warp] = it;
        wp[warp] = ip;
    }
    __syncthreads();  // (s_bad is 0 by now)
    if (bad) s_bad = 1;
    if (warp == 0) {
        long long x = wt[lane], y = wp[lane];
        const long long x0 = x, y0 = y;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long u = __shfl_up_sync(~0u, x, d), v = __shfl_up_sync(~0u, y, d);
            if (lane >= d) {
                x += u;
                y += v;
            }
        }
        if (lane == 31) {
            s_tot[0] = x;
            s_tot[1] = y;
        }
        wt[lane] = x - x0;
        wp[lane] = y - y0;
    }
    __syncthreads();
    const long long tokens = s_tot[0], pages = s_tot[1];
    int code = KG_OK;
    if (s_bad || tokens > a.max_tokens) code = KG_ERR_INVALID_ARG;
    else if (pages > nf) code = KG_ERR_OOM;
    if (code == KG_OK) {
        long long bt = wt[warp] + it - t, bp = wp[warp] + ip - p;
        for (int r = r0; r < r1; ++r) {
            const int n = a.fresh[r];
            const long long c = old[r];
            cu[r] = (int)bt;
            pg[r] = (int)bp;
            bt += n;
            bp += pages_of(c + n, shift) - pages_of(c, shift);
        }
        if (tid == 0) {
            cu[a.n_req] = (int)tokens;
            pg[a.n_req] = (int)pages;
        }
        for (int i = gid; i < (int)pages; i += step) {
            const int e = a.free_pages[nf - 1 - i];
            if (e < 0 || e >= a.n_pages) s_bad = 1;
        }
    }
    __syncthreads();
    if (ctas > 1) {  // every CTA has read the free count and checked its share; nothing has been written
        asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;\n" ::: "memory");
        int other = 0;
        if (lane < (int)ctas) {
            uint32_t at;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(&s_bad)), "r"(lane));
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(other) : "r"(at) : "memory");
        }
        if (__any_sync(~0u, other != 0)) code = KG_ERR_INVALID_ARG;
        asm volatile("barrier.cluster.arrive.release;\n" ::: "memory");  // (waited for at the end: no CTA leaves before it has been read)
    } else if (s_bad) {
        code = KG_ERR_INVALID_ARG;
    }
    if (gid == 0) {
        *a.status = code;
        *a.n_free_out = code == KG_OK ? nf - (int)pages : nf;
    }
    if (code != KG_OK) {  // the step does nothing
        for (int r = gid; r <= a.n_req; r += step) a.cu[r] = 0;
        for (int r = gid; r < a.n_req; r += step) a.kv[r] = 0;
        for (uint32_t i = gid; i < (uint32_t)a.max_tokens; i += step) a.slots[i] = a.req[i] = a.pos[i] = -1;
    } else {
        for (int r = gid; r <= a.n_req; r += step) a.cu[r] = cu[r];
        for (int r = gid; r < a.n_req; r += step) a.kv[r] = old[r] + cu[r + 1] - cu[r];
        for (int i = gid; i < (int)pages; i += step) {
            const int r = range_of(pg, a.n_req, i);
            a.table[(int64_t)r * a.width + pages_of(old[r], shift) + i - pg[r]] = a.free_pages[nf - 1 - i];
        }
#pragma unroll 4
        for (uint32_t i = gid; i < (uint32_t)a.max_tokens; i += step) {  // (i may pass 2^31 by a step)
            int slot = -1, r = -1, x = -1;
            if (i < (uint32_t)tokens) {
                r = range_of(cu, a.n_req, (int)i);
                const int c = old[r];
                x = c + (int)i - cu[r];
                const int has = pages_of(c, shift), q = x >> shift;
                const int e = __ldg(q < has ? a.table + (int64_t)r * a.width + q : a.free_pages + (nf - 1 - (pg[r] + q - has)));
                slot = (e << shift) + (x & (a.page - 1));
            }
            a.slots[i] = slot;
            a.req[i] = r;
            a.pos[i] = x;
        }
    }
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire;\n" ::: "memory");
}

// ---------------------------------------------------------------------------
// Store: one thread moves eight elements of one row, K or V: 16 bytes written, 16 or
// 32 read, neighbours side by side on both sides. 256 rows of 32 heads of 128: 2.6 us in a
// graph, 8.8 us a call, the host's time. Bound by HBM beyond: 16,500 f32 rows of 12
// heads of 64, 151 MB, in 27 us (85% of the copy rate).
struct StoreArgs {
    kg_pool p;
    const void *k, *v;
    int64_t row_stride, head_stride;
    const int32_t *slots;
    int n_rows, places;
    int *err;
};

template <typename D>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

template <typename S>
__device__ __forceinline__ void load8(const S *p, float (&f)[8]) {
    alignas(16) S x[8];
#pragma unroll
    for (int i = 0; i < (int)sizeof(x) / 16; ++i)
        reinterpret_cast<uint4 *>(x)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f(x[i]);
}

template <typename S, typename D>
__global__ void __launch_bounds__(256) store_kernel(StoreArgs a) {
    pdl_wait();
    const int per_head = a.p.head_dim / 8, per_row = a.p.n_kv_head * per_head;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.n_rows * per_row) return;
    const int row = (int)(i / per_row), c = (int)(i % per_row), h = c / per_head, d = (c % per_head) * 8;
    const int slot = a.slots[row];
    if (slot < 0) return;
    if (slot >= a.places) {
        if (c == 0 && blockIdx.y == 0) reject(a.err);
        return;
    }
    const S *src = static_cast<const S *>(blockIdx.y ? a.v : a.k) + row * a.row_stride + h * a.head_stride + d;
    D *dst = static_cast<D *>(blockIdx.y ? a.p.v : a.p.k) + (slot / a.p.page_size) * a.p.page_stride +
             (slot % a.p.page_size) * a.p.row_stride + h * a.p.head_stride + d;
    float f[8];
    load8(src, f);
    *reinterpret_cast<uint4 *>(dst) =
        make_uint4(pack2<D>(f[0], f[1]), pack2<D>(f[2], f[3]), pack2<D>(f[4], f[5]), pack2<D>(f[6], f[7]));
}

template <typename S>
cudaError_t launch_store(const StoreArgs &a, cudaStream_t s) {
    const int64_t n = (int64_t)a.n_rows * a.p.n_kv_head * (a.p.head_dim / 8);
    const dim3 grid((unsigned)((n + 255) / 256), 2);
    if (a.p.dtype == KG_DT_BF16) return launch_pdl(store_kernel<S, __nv_bfloat16>, grid, dim3(256), 0, s, a);
    return launch_pdl(store_kernel<S, __half>, grid, dim3(256), 0, s, a);
}

}  // namespace
}  // namespace serve
}  // namespace kg

extern "C" {

int kg_pool_plan_dev(kg_ctx *ctx, int32_t page_size, int32_t n_pages, int32_t n_req, const int32_t *cached_len,
                     const int32_t *new_len, int32_t *table, int32_t table_width, const int32_t *free_pages,
                     const int32_t *n_free, int32_t *n_free_out, int32_t max_tokens, int32_t *cu_q, int32_t *kv_len,
                     int32_t *slots, int32_t *req_of, int32_t *positions, int32_t *status, void *stream) {
    using namespace kg::serve;
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
        return fail(ctx, KG_ERR_UNSUPPORTED, "plan: page_size must be 16, 32, 64 or 128");
    if (n_pages < 1 || (int64_t)n_pages * page_size > INT32_MAX)
        return fail(ctx, KG_ERR_INVALID_ARG, "plan: n_pages must be positive and n_pages * page_size below 2^31");
    if (n_req < 0 || table_width < 1 || max_tokens < 0)
        return fail(ctx, KG_ERR_INVALID_ARG, "plan: n_req and max_tokens must not be negative, table_width positive");
    if (n_req > kMaxReq) return fail(ctx, KG_ERR_UNSUPPORTED, "plan: at most 16384 requests");
    if (!n_free || !n_free_out || !cu_q || !status || !free_pages ||
        (n_req > 0 && (!cached_len || !new_len || !table || !kv_len)) || (max_tokens > 0 && (!slots || !req_of || !positions)))
        return fail(ctx, KG_ERR_INVALID_ARG, "plan: null pointer");
    if (!ctx) return fail(ctx, KG_ERR_INVALID_ARG, "null context");
    DeviceGuard dg(ctx->device);
    if (dg.err != cudaSuccess) return cuda_fail(ctx, dg.err, "kg_pool_plan_dev");
    PlanArgs a{page_size, n_pages, n_req, table_width, max_tokens, cached_len, new_len, table, free_pages,
               n_free, n_free_out, cu_q, kv_len, slots, req_of, positions, status};
    const size_t smem = (size_t)(3 * n_req + 2) * sizeof(int32_t);
    const int ctas = max_tokens > 2 * PLAN_THREADS || n_req > 2 * PLAN_THREADS ? 8 : 1;
    cudaError_t e = smem > 40 * 1024 ? kg::dev::smem(plan_kernel, smem) : cudaSuccess;
    if (e == cudaSuccess)
        e = kg::launch_pdl_cluster(plan_kernel, dim3(ctas), dim3(PLAN_THREADS), smem, static_cast<cudaStream_t>(stream), dim3(ctas), a);
    return e == cudaSuccess ? KG_OK : cuda_fail(ctx, e, "kg_pool_plan_dev");
}

int kg_pool_store_dev(kg_ctx *ctx, const kg_pool *pool, int32_t n_rows, const int32_t *slots, int32_t src_dtype,
                      const void *k, const void *v, int64_t row_stride, int64_t head_stride, void *stream) {
    using namespace kg::serve;
    if (int rc = check_pool(ctx, pool)) return rc;
    if (n_rows < 0) return fail(ctx, KG_ERR_INVALID_ARG, "store: n_rows must not be negative");
    if (src_dtype != KG_DT_F32 && src_dtype != KG_DT_BF16 && src_dtype != KG_DT_F16)
        return fail(ctx, KG_ERR_UNSUPPORTED, "store: src_dtype must be KG_DT_F32, KG_DT_BF16 or KG_DT_F16");
    if ((int64_t)n_rows * pool->n_kv_head > INT32_MAX) return fail(ctx, KG_ERR_UNSUPPORTED, "store: too many rows (n_rows * n_kv_head)");
    if (n_rows > 0) {
        if (!slots || !k || !v) return fail(ctx, KG_ERR_INVALID_ARG, "store: null pointer");
        const int unit = src_dtype == KG_DT_F32 ? 4 : 8;
        if (!aligned16(k) || !aligned16(v) || row_stride % unit || head_stride % unit || row_stride < 0 || head_stride < 0)
            return fail(ctx, KG_ERR_INVALID_ARG, "store: rows must be 16-byte aligned, strides not negative");
    }
    if (!ctx) return fail(ctx, KG_ERR_INVALID_ARG, "null context");
    if (n_rows == 0) return KG_OK;
    DeviceGuard dg(ctx->device);
    if (dg.err != cudaSuccess) return cuda_fail(ctx, dg.err, "kg_pool_store_dev");
    StoreArgs a{*pool, k, v, row_stride, head_stride, slots, n_rows, pool->n_pages * pool->page_size, ctx->serve_err};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = src_dtype == KG_DT_F32    ? launch_store<float>(a, s)
                          : src_dtype == KG_DT_BF16 ? launch_store<__nv_bfloat16>(a, s)
                                                    : launch_store<__half>(a, s);
    return e == cudaSuccess ? KG_OK : cuda_fail(ctx, e, "kg_pool_store_dev");
}

int kg_pool_status(kg_ctx *ctx) {
    using namespace kg::serve;
    if (!ctx) return fail(ctx, KG_ERR_INVALID_ARG, "null context");
    DeviceGuard dg(ctx->device);
    cudaError_t e = dg.err;
    int word = 0;
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(&word, ctx->serve_err, sizeof(word), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && word) e = cudaMemset(ctx->serve_err, 0, sizeof(word));
    if (e != cudaSuccess) return cuda_fail(ctx, e, "kg_pool_status");
    if (word == KG_ERR_TIMEOUT) return fail(ctx, KG_ERR_TIMEOUT, "a device-side wait exceeded its limit");
    if (word) return fail(ctx, KG_ERR_INVALID_ARG, "device rejected a length, slot or table entry of a kg_pool call");
    return KG_OK;
}

}  // extern "C"
