// kg_logits.cu — kg_sample_logits_dev: next tokens from logits with top-k,
// top-p and min-p, every row with its own parameters and its own uniform number.
//
// A row is ordered by (value descending, index ascending). Weights are
// w = exp((x - max) / T) rounded to integer units of 2^-44, so that every sum
// is exact whatever its order and a comparison next to a border comes out the
// same on every run: a rounding is 2^-45 of the largest weight, against the
// 2^-24 spacing of the given uniform numbers. Every cut of the order is a key
// (the value's bits in order) and an index: a token stays if its key is above
// the cut's, or equal with an index below the cut's.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kg_pdl.cuh"
#include "kg_serve.h"

namespace kg {
namespace serve {
namespace {

typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    int64_t ld;
    int n_rows, vocab;
    const float *temp;
    const int32_t *top_k;
    const float *top_p, *min_p, *u;
    int32_t *out;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

// the value's bits as an unsigned number in the values' order; 0 for what is
// never drawn (-inf, NaN); -0 counts as +0
__device__ __forceinline__ uint32_t key_of(float x) {
    x += 0.0f;
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

constexpr int THREADS = 1024;
constexpr double UNIT = 17592186044416.0;  // 2^44

__device__ u64 block_sum(u64 v, u64 *tmp) {
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < THREADS / 32; ++w) v += tmp[w];
    return v;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_logits_kernel(SampleArgs a) {
    pdl_wait();
    __shared__ u64 tmp[THREADS / 32];
    const int row = blockIdx.x, V = a.vocab, tid = threadIdx.x;
    const T *x = static_cast<const T *>(a.logits) + row * a.ld;
    // sum over the row of f(key, index)
    auto total = [&](auto f) {
        u64 s = 0;
        for (int j = tid; j < V; j += THREADS) s += f(key_of(to_f(x[j])), (uint32_t)j);
        return block_sum(s, tmp);
    };
    // the largest c whose sum over keys >= c reaches `want` (> 0)
    auto cut_key = [&](u64 want, auto f) {
        uint32_t c = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
            const uint32_t t = c | bit;
            if (total([&](uint32_t k, uint32_t j) { return k >= t ? f(k, j) : 0ull; }) >= want) c = t;
        }
        return c;
    };
    // the smallest n whose sum over indexes < n reaches `want` (> 0)
    auto cut_index = [&](u64 want, auto f) {
        uint32_t lo = 0, hi = V;  // sum(< lo) < want <= sum(< hi)
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (total([&](uint32_t k, uint32_t j) { return j < mid ? f(k, j) : 0ull; }) >= want) hi = mid;
            else lo = mid;
        }
        return hi;
    };
    const u64 live = total([](uint32_t k, uint32_t) { return k ? 1ull : 0ull; });
    if (live == 0) {
        if (tid == 0) a.out[row] = -1;
        return;
    }
    const uint32_t kmax = cut_key(1, [](uint32_t, uint32_t) { return 1ull; });
    const float T_ = a.temp ? a.temp[row] : 1.0f;
    if (!(T_ > 0.0f)) {
        const uint32_t n = cut_index(1, [&](uint32_t k, uint32_t) { return k == kmax ? 1ull : 0ull; });
        if (tid == 0) a.out[row] = (int)n - 1;
        return;
    }
    const float xmax = value_of(kmax), mp = a.min_p && a.min_p[row] > 0.0f ? fminf(a.min_p[row], 1.0f) : 0.0f;
    auto weight_f = [&](uint32_t k) -> double {
        if (k == kmax) return 1.0;
        const float xv = value_of(k);
        if (isinf(xmax)) return 0.0;
        return exp(((double)xv - (double)xmax) / (double)T_);
    };
    auto weight = [&](uint32_t k) -> u64 { return k ? (u64)__double2ll_rn(weight_f(k) * UNIT) : 0ull; };
    uint32_t ck = 1, ci = V;  // the cut
    auto stays = [&](uint32_t k, uint32_t j) { return k > ck || (k == ck && j < ci); };
    const int want_k = a.top_k ? a.top_k[row] : 0;
    if (want_k > 0 && (u64)want_k < live) {
        const uint32_t c = cut_key(want_k, [](uint32_t k, uint32_t) { return k ? 1ull : 0ull; });
        const u64 above = total([&](uint32_t k, uint32_t) { return k > c ? 1ull : 0ull; });
        ci = cut_index(want_k - above, [&](uint32_t k, uint32_t) { return k == c ? 1ull : 0ull; });
        ck = c;
    }
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    if (p < 1.0f) {
        auto mass = [&](uint32_t k, uint32_t j) { return stays(k, j) ? weight(k) : 0ull; };
        const u64 W = total(mass);
        const double t = ceil((double)fmaxf(p, 0.0f) * (double)W);
        const u64 want = t < 1.0 ? 1ull : (u64)t;
        const uint32_t c = cut_key(want, mass);
        const u64 above = total([&](uint32_t k, uint32_t j) { return k > c ? mass(k, j) : 0ull; });
        const u64 w = weight(c), m = (want - above + w - 1) / w;
        const uint32_t n = cut_index(m, [&](uint32_t k, uint32_t j) { return k == c && stays(k, j) ? 1ull : 0ull; });
        ck = c;
        ci = n;
    }
    auto kept = [&](uint32_t k, uint32_t j) -> u64 {
        if (!k || !stays(k, j)) return 0;
        const double w = weight_f(k);
        return w < (double)mp ? 0ull : (u64)__double2ll_rn(w * UNIT);
    };
    const u64 K = total(kept);
    const double u = a.u[row] > 0.0f ? (double)a.u[row] : 0.0;
    u64 t = u >= 1.0 ? K - 1 : (u64)(u * (double)K);
    if (t > K - 1) t = K - 1;
    const uint32_t n = cut_index(t + 1, kept);  // running sum > t
    if (tid == 0) a.out[row] = (int)n - 1;
}

}  // namespace
}  // namespace serve
}  // namespace kg

extern "C" int kg_sample_logits_dev(kg_ctx *ctx, int32_t n_rows, int32_t vocab, int32_t dtype, const void *logits,
                                    int64_t ld, const float *temperature, const int32_t *top_k, const float *top_p,
                                    const float *min_p, const float *u, int32_t *tokens_out, void *stream) {
    using namespace kg::serve;
    if (n_rows < 0 || vocab < 1) return fail(ctx, KG_ERR_INVALID_ARG, "sample: n_rows must not be negative, vocab positive");
    if (vocab > kMaxVocab) return fail(ctx, KG_ERR_UNSUPPORTED, "sample: vocab at most 262144");
    if (dtype != KG_DT_F32 && dtype != KG_DT_BF16 && dtype != KG_DT_F16)
        return fail(ctx, KG_ERR_UNSUPPORTED, "sample: dtype must be KG_DT_F32, KG_DT_BF16 or KG_DT_F16");
    if (n_rows > 0 && (!logits || !u || !tokens_out)) return fail(ctx, KG_ERR_INVALID_ARG, "sample: null pointer");
    if (n_rows > 1 && ld < vocab) return fail(ctx, KG_ERR_INVALID_ARG, "sample: rows overlap (ld < vocab)");
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == KG_DT_F32 ? 4 : 2))
        return fail(ctx, KG_ERR_INVALID_ARG, "sample: logits not aligned to their type");
    if (!ctx) return fail(ctx, KG_ERR_INVALID_ARG, "null context");
    if (n_rows == 0) return KG_OK;
    DeviceGuard dg(ctx->device);
    if (dg.err != cudaSuccess) return cuda_fail(ctx, dg.err, "kg_sample_logits_dev");
    SampleArgs a{logits, n_rows > 1 ? ld : 0, n_rows, vocab, temperature, top_k, top_p, min_p, u, tokens_out};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const dim3 grid(n_rows), block(THREADS);
    const cudaError_t e = dtype == KG_DT_F32    ? kg::launch_pdl(sample_logits_kernel<float>, grid, block, 0, s, a)
                          : dtype == KG_DT_BF16 ? kg::launch_pdl(sample_logits_kernel<__nv_bfloat16>, grid, block, 0, s, a)
                                                : kg::launch_pdl(sample_logits_kernel<__half>, grid, block, 0, s, a);
    return e == cudaSuccess ? KG_OK : cuda_fail(ctx, e, "kg_sample_logits_dev");
}
