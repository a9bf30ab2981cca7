// kg_logits.cu — kg_sample_logits_dev: next tokens from logits with top-k,
// top-p and min-p, every row with its own parameters and its own uniform number.
//
// A row is ordered by (value descending, index ascending). Weights are
// w = 2^((x - max) log2(e) / T) in integer units of 2^-44, so that every sum is
// exact whatever its order and a comparison next to a border comes out the same on
// every run: a rounding is 2^-45 of the largest weight, against the 2^-24 spacing
// of the given uniform numbers. Every cut of the order is a key (the value's bits in
// order) and an index: a token stays if its key is above the cut's, or equal with an
// index below the cut's.
//
// A row is held in the shared memory of a cluster of 1 to 8 CTAs and read from
// global memory once. A histogram of (max - x) / T in steps of 1/64 says where the
// cuts must lie:
//   - where the candidates down to that step are at most 512 (small top-k, a peaked
//     row), they go to the cluster's first CTA, which ranks and cuts them alone;
//   - else the tokens of the step (top-k) or of three steps (top-p) that hold the cut
//     go there, at most 4096, and the cut is found by bisection of their keys against
//     the exact sum above them; the token is drawn by all CTAs;
//   - where that does not hold (rows of equal values), by bisection over the row.
// Weights cost about 12 operations in 64 bits: they are computed for what a sum needs.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kg_dev.cuh"
#include "kg_pdl.cuh"
#include "kg_serve.h"

namespace kg {
namespace serve {
namespace {

typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    int64_t ld;
    int n_rows, vocab, slice;  // slice: entries of a CTA
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

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 2048, LOCAL = 512, LIST = 4096;
static_assert(LOCAL == THREADS, "a thread has one candidate");

// ---- cluster
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;\n" ::: "memory");
}
// address of `p` (shared memory of this CTA) in CTA `rank`
__device__ __forceinline__ uint32_t remote(const void *p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ uint32_t remote_u32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ u64 remote_u64(uint32_t a) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void remote_store(uint32_t a, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
__device__ __forceinline__ uint32_t remote_add(uint32_t a, uint32_t v) {
    uint32_t r;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(a), "r"(v) : "memory");
    return r;
}

struct Shared {
    double tab[64];        // 2^(j / 64)
    u64 warp[2][WARPS];    // block sums
    u64 red[2];            // this CTA's part of a cluster sum
    u64 cut;               // (key << 32 | index) found by the first CTA
    uint32_t n_list, wanted[2];
    int32_t found;
    union {
        struct {
            uint32_t hist[BINS], sum[BINS];  // this CTA's counts, the cluster's
        };
        u64 list[LIST];  // key << 32 | index, of the first CTA
    };
};

// The weight's arithmetic: 2^y by a table of 2^(j / 64) and the series of 2^r, |r| <= 1/128 (the first term left out is
// below 2^-54).
struct Weigh {
    double c, xmax;  // log2(e) / T
    uint32_t kmax;
    bool inf;
    const double *tab;
    __device__ __forceinline__ double real(uint32_t k) const {  // in units
        if (k == kmax) return 17592186044416.0;
        const double y = ((double)value_of(k) - xmax) * c;
        if (inf || !(y > -46.0)) return 0.0;
        const double t = fma(y, 64.0, 6755399441055744.0);  // rounds to an integer in the low bits
        const int n = __double2loint(t);
        const double r = fma(t - 6755399441055744.0, -0.015625, y);
        double p = 0.00133335581464284434;  // ln(2)^n / n!
        p = fma(p, r, 0.00961812910762847716);
        p = fma(p, r, 0.0555041086648215800);
        p = fma(p, r, 0.240226506959100712);
        p = fma(p, r, 0.693147180559945309);
        p = fma(p, r, 1.0);
        p *= tab[n & 63];
        return __hiloint2double(__double2hiint(p) + (((n >> 6) + 44) << 20), __double2loint(p));
    }
    static __device__ __forceinline__ u64 whole(double w) {  // w below 2^51, to the nearest
        return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 operator()(uint32_t k) const { return k ? whole(real(k)) : 0ull; }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) sample_logits_kernel(SampleArgs a) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared &sh = *reinterpret_cast<Shared *>(raw);
    uint32_t *keys = reinterpret_cast<uint32_t *>(raw + sizeof(Shared));
    const uint32_t rank = cluster_rank(), C = cluster_size();
    const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int base = (int)rank * a.slice, n = max(0, min(a.slice, a.vocab - base));
    if (tid < 64) sh.tab[tid] = exp2(tid / 64.0);
    pdl_wait();
    const float T_ = a.temp ? a.temp[row] : 1.0f, p = a.top_p ? a.top_p[row] : 1.0f;
    const float mp = a.min_p && a.min_p[row] > 0.0f ? fminf(a.min_p[row], 1.0f) : 0.0f;
    const int want_k = a.top_k ? a.top_k[row] : 0;
    const float u_in = a.u[row];

    int flip = 0;  // sums in turn use two places: one is read while the next is written
    auto block_sum = [&](u64 v) {
        v = warp_sum(v);
        u64 *w = sh.warp[flip & 1];
        ++flip;
        if (lane == 0) w[warp] = v;
        __syncthreads();
        v = lane < WARPS ? w[lane] : 0;
        return warp_sum(v);
    };
    int turn = 0;
    // every CTA's v (the same in all its threads): f(rank, v)
    auto gather = [&](u64 v, auto f) {
        if (tid == 0) sh.red[turn & 1] = v;
        cluster_sync();
        for (uint32_t r = 0; r < C; ++r) f(r, remote_u64(remote(&sh.red[turn & 1], r)));
        ++turn;
    };
    auto cluster_sum = [&](u64 v) {
        u64 s = 0;
        gather(block_sum(v), [&](uint32_t, u64 x) { s += x; });
        return s;
    };

    // the row's slice into shared memory, as keys
    uint32_t top = 0;
    {
        const T *x = static_cast<const T *>(a.logits) + row * a.ld + base;
        constexpr int W = 16 / sizeof(T);
        const int head = (int)min((uintptr_t)n, ((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));
        const int vecs = (n - head) / W, tail = head + vecs * W;
        auto put = [&](int i, float v) {
            const uint32_t k = key_of(v);
            keys[i] = k;
            top = max(top, k);
        };
        if (tid < head) put(tid, to_f(x[tid]));
#pragma unroll 4
        for (int i = tid; i < vecs; i += THREADS) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(x + head) + i);
            const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
            for (int k = 0; k < W; ++k) put(head + i * W + k, to_f(e[k]));
        }
        if (tail + tid < n) put(tail + tid, to_f(x[tail + tid]));
    }
    top = __reduce_max_sync(~0u, top);
    if (lane == 0) sh.warp[0][warp] = top;
    __syncthreads();
    top = __reduce_max_sync(~0u, lane < WARPS ? (uint32_t)sh.warp[0][lane] : 0u);
    flip = 1;
    uint32_t kmax = 0;
    gather(top, [&](uint32_t, u64 x) { kmax = max(kmax, (uint32_t)x); });

    // the smallest index (of the row) that any thread of the cluster names
    auto first_index = [&](uint32_t mine) {
        mine = __reduce_min_sync(~0u, mine);
        u64 *w = sh.warp[flip & 1];
        ++flip;
        if (lane == 0) w[warp] = mine;
        __syncthreads();
        mine = __reduce_min_sync(~0u, lane < WARPS ? (uint32_t)w[lane] : ~0u);
        uint32_t all = ~0u;
        gather(mine, [&](uint32_t, u64 x) { all = min(all, (uint32_t)x); });
        return all;
    };
    auto done = [&](int token) {  // (no CTA leaves while another may read its shared memory)
        if (rank == 0 && tid == 0) a.out[row] = token;
        cluster_sync();
    };
    if (kmax == 0) return done(-1);
    if (!(T_ > 0.0f)) {
        uint32_t at = ~0u;
        for (int i = tid; i < n; i += THREADS)
            if (keys[i] == kmax) at = min(at, (uint32_t)(base + i));
        return done((int)first_index(at));
    }
    Weigh weigh{1.4426950408889634 / (double)T_, (double)value_of(kmax), kmax, isinf(value_of(kmax)) != 0, sh.tab};
    const double mp_units = (double)mp * 17592186044416.0;
    const float xmax = value_of(kmax), step = 64.0f / T_;
    auto bin_of = [&](uint32_t k) { return k == kmax ? 0 : min(BINS - 1, (int)((xmax - value_of(k)) * step)); };

    uint32_t ck = 1, ci = ~0u;  // the cut
    auto stays = [&](uint32_t k, uint32_t j) { return k > ck || (k == ck && j < ci); };
    auto over = [&](auto f) {  // sum over the row of f(key, index)
        u64 s = 0;
        for (int i = tid; i < n; i += THREADS) s += f(keys[i], (uint32_t)(base + i));
        return cluster_sum(s);
    };
    // Bisection over the row: the largest key whose sum over keys >= it reaches `want`, and the smallest count of its
    // first equals that does.
    auto cut_row = [&](u64 want, auto f, auto per_equal) {
        uint32_t c = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
            const uint32_t t = c | bit;
            if (over([&](uint32_t k, uint32_t j) { return k >= t ? f(k, j) : 0ull; }) >= want) c = t;
        }
        const u64 above = over([&](uint32_t k, uint32_t j) { return k > c ? f(k, j) : 0ull; });
        const u64 w = per_equal(c), m = (want - above + w - 1) / w;
        uint32_t lo = 0, hi = a.vocab;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (over([&](uint32_t k, uint32_t j) { return k == c && j < mid && stays(k, j) ? 1ull : 0ull; }) >= m) hi = mid;
            else lo = mid;
        }
        ck = c;
        ci = hi;
    };
    // The same over the first CTA's list; the cut goes to every CTA.
    auto cut_list = [&](u64 want, auto f, auto per_equal) {
        if (rank == 0) {
            const int m = (int)sh.n_list;
            auto sum = [&](auto g) {
                u64 s = 0;
                for (int i = tid; i < m; i += THREADS) {
                    const u64 e = sh.list[i];
                    s += g((uint32_t)(e >> 32), (uint32_t)e);
                }
                return block_sum(s);
            };
            uint32_t lo = 0, hi = 0;  // keys that the list's share the leading bits of
            {
                uint32_t x = 0, y = ~0u;
                for (int i = tid; i < m; i += THREADS) {
                    const uint32_t k = (uint32_t)(sh.list[i] >> 32);
                    x = max(x, k);
                    y = min(y, k);
                }
                x = __reduce_max_sync(~0u, x);
                y = __reduce_min_sync(~0u, y);
                u64 *w = sh.warp[flip & 1];
                ++flip;
                if (lane == 0) w[warp] = (u64)x << 32 | y;
                __syncthreads();
                hi = __reduce_max_sync(~0u, lane < WARPS ? (uint32_t)(w[lane] >> 32) : 0u);
                lo = __reduce_min_sync(~0u, lane < WARPS ? (uint32_t)w[lane] : ~0u);
            }
            while (lo < hi) {  // sum(>= lo) reaches want; the cut is in [lo, hi]
                const uint32_t mid = lo + (hi - lo + 1) / 2;
                if (sum([&](uint32_t k, uint32_t j) { return k >= mid ? f(k, j) : 0ull; }) >= want) lo = mid;
                else hi = mid - 1;
            }
            const uint32_t c = lo;
            const u64 above = sum([&](uint32_t k, uint32_t j) { return k > c ? f(k, j) : 0ull; });
            const u64 w = per_equal(c), take = (want - above + w - 1) / w;
            const u64 have = sum([&](uint32_t k, uint32_t j) { return k == c && stays(k, j) ? 1ull : 0ull; });
            uint32_t at = ~0u;  // all of the equals
            if (take < have) {
                uint32_t l = 0;
                at = a.vocab;
                while (at - l > 1) {
                    const uint32_t mid = (l + at) / 2;
                    if (sum([&](uint32_t k, uint32_t j) { return k == c && j < mid && stays(k, j) ? 1ull : 0ull; }) >= take) at = mid;
                    else l = mid;
                }
            }
            if (tid == 0) sh.cut = (u64)c << 32 | at;
        }
        cluster_sync();
        const u64 x = remote_u64(remote(&sh.cut, 0));
        const uint32_t ci_before = ci, ck_before = ck;
        ck = (uint32_t)(x >> 32);
        ci = (uint32_t)x;
        if (ck == ck_before) ci = min(ci, ci_before);
    };
    // live entries whose bin is in [b0, b1] into the first CTA's list (only what stays)
    auto to_list = [&](int b0, int b1) {
        if (tid == 0) sh.n_list = 0;
        cluster_sync();  // (and the histograms, which lie under the list, have been read)
        const uint32_t count = remote(&sh.n_list, 0), dst = remote(sh.list, 0);
        for (int i0 = 0; i0 < n; i0 += THREADS) {
            const int i = i0 + tid;
            const uint32_t k = i < n ? keys[i] : 0u;
            bool in = k != 0;
            if (in) {
                const int b = bin_of(k);
                in = b >= b0 && b <= b1 && stays(k, (uint32_t)(base + i));
            }
            const uint32_t who = __ballot_sync(~0u, in);
            if (who == 0) continue;
            uint32_t at = 0;
            if (lane == __ffs(who) - 1) at = remote_add(count, __popc(who));
            at = __shfl_sync(~0u, at, __ffs(who) - 1) + __popc(who & ((1u << lane) - 1));
            if (in && at < LIST) remote_store(dst + at * 8, (u64)k << 32 | (uint32_t)(base + i));
        }
        cluster_sync();
    };

    const u64 kk = want_k > 0 && want_k < a.vocab ? (u64)want_k : 0ull;
    if (kk || p < 1.0f) {
        // counts by bin, and where no top-k precedes it the whole sum for top-p
        for (int i = tid; i < BINS; i += THREADS) sh.hist[i] = 0;
        __syncthreads();
        u64 mine = 0;
        const bool mass = p < 1.0f && !kk;
        for (int i = tid; i < n; i += THREADS) {
            const uint32_t k = keys[i];
            if (k == 0) continue;
            atomicAdd(&sh.hist[bin_of(k)], 1u);
            if (mass) mine += weigh(k);
        }
        u64 W = cluster_sum(mine);  // (synchronises: every histogram is complete)
        uint32_t cnt[BINS / THREADS];
        const int b0 = tid * (BINS / THREADS);
        for (int j = 0; j < BINS / THREADS; ++j) cnt[j] = 0;
        for (uint32_t r = 0; r < C; ++r) {
            const uint32_t h = remote(&sh.hist[b0], r);
            for (int j = 0; j < BINS / THREADS; ++j) cnt[j] += remote_u32(h + j * 4);
        }
        // running sums of counts and of estimated weights over the bins
        auto scan = [&](u64 v) {  // exclusive, over the block's threads
            u64 x = v;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const u64 y = __shfl_up_sync(~0u, x, d);
                if (lane >= d) x += y;
            }
            u64 *w = sh.warp[flip & 1];
            ++flip;
            if (lane == 31) w[warp] = x;
            __syncthreads();
            u64 before = 0;
            for (int k = 0; k < warp; ++k) before += w[k];
            return before + x - v;
        };
        u64 c_here = 0, e_here = 0;
        auto guess = [&](int b) { return (u64)(exp2f((b + 0.5f) * (-1.44269504f / 64.0f)) * 1073741824.0f) + 1; };
        for (int j = 0; j < BINS / THREADS; ++j) {
            c_here += cnt[j];
            e_here += cnt[j] * guess(b0 + j);
        }
        u64 c_run = scan(c_here), e_run = scan(e_here);
        const u64 live = block_sum(c_here), e_all = block_sum(e_here);
        const bool use_k = kk && kk < live;
        if (kk && !use_k && p < 1.0f) W = over([&](uint32_t k, uint32_t) { return weigh(k); });
        // the bin of the k-th entry, the bin where top-p's cut is expected, and the counts down to them
        const u64 e_want = (u64)((double)fmaxf(p, 0.0f) * (double)e_all);
        if (tid == 0) sh.wanted[0] = sh.wanted[1] = BINS - 1;
        __syncthreads();
        for (int j = 0; j < BINS / THREADS; ++j) {
            const u64 e = cnt[j] * guess(b0 + j);
            if (use_k && c_run < kk && kk <= c_run + cnt[j]) sh.wanted[0] = b0 + j;
            if (e_run <= e_want && e_want < e_run + e) sh.wanted[1] = b0 + j;
            sh.sum[b0 + j] = (uint32_t)(c_run += cnt[j]);  // entries in bins <= b
            e_run += e;
        }
        __syncthreads();
        const int bk = (int)sh.wanted[0], bp = (int)sh.wanted[1];
        auto upto = [&](int b) { return b < 0 ? 0u : sh.sum[b]; };
        const uint32_t n_local = upto(use_k ? bk : min(bp + 1, BINS - 1));
        const uint32_t n_k = use_k ? upto(bk) - upto(bk - 1) : 0u;
        const u64 k_left = use_k ? kk - upto(bk - 1) : 0ull;
        const int p0 = max(bp - 1, 0), p1 = min(bp + 1, BINS - 1);
        const uint32_t n_p = upto(p1) - upto(p0 - 1);
        if (n_local <= LOCAL && (use_k || p < 1.0f)) {
            // Few candidates: the first CTA ranks them in both orders and finishes the row.
            to_list(0, use_k ? bk : p1);
            if (rank == 0) {
                const int m = (int)sh.n_list;
                u64 *by_order = sh.list + LOCAL;                                      // weights in order
                uint32_t *place = reinterpret_cast<uint32_t *>(sh.list + 2 * LOCAL);  // by index: place in the order, then the index
                __syncthreads();
                if (tid < m) {
                    const u64 e = sh.list[tid];
                    const uint32_t k = (uint32_t)(e >> 32), j = (uint32_t)e;
                    int ro = 0, ri = 0;
#pragma unroll 4
                    for (int q = 0; q < m; ++q) {
                        const u64 x = sh.list[q];
                        const uint32_t xk = (uint32_t)(x >> 32), xj = (uint32_t)x;
                        ri += xj < j;
                        ro += xk > k || (xk == k && xj < j);
                    }
                    by_order[ro] = weigh(k);
                    place[ri] = ro | (weigh.real(k) < mp_units ? 0x80000000u : 0u);
                    place[LOCAL + ri] = j;
                }
                __syncthreads();
                u64 w = tid < m && (!use_k || (u64)tid < kk) ? by_order[tid] : 0ull;
                u64 run = scan(w);
                const u64 sum = block_sum(w);
                if (use_k) W = sum;  // what top-k leaves
                const double t = ceil((double)fmaxf(p, 0.0f) * (double)W);
                const u64 want = p < 1.0f ? (t < 1.0 ? 1ull : (u64)t) : ~0ull;
                if (tid == 0) sh.found = p < 1.0f && sum < want ? -2 : -1;  // -2: the cut lies behind the list
                if (tid < m) by_order[tid] = run < want ? w : 0ull;  // stays where what precedes it has not reached the whole
                __syncthreads();
                if (sh.found != -2) {
                    const uint32_t q = tid < m ? place[tid] : 0x80000000u;
                    w = q & 0x80000000u ? 0ull : by_order[q];
                    run = scan(w);
                    const u64 K = block_sum(w);
                    const double uu = u_in > 0.0f ? (double)u_in : 0.0;
                    u64 tt = uu >= 1.0 ? K - 1 : (u64)(uu * (double)K);
                    if (tt > K - 1) tt = K - 1;
                    if (run <= tt && tt < run + w) sh.found = (int)place[LOCAL + tid];
                }
                __syncthreads();
            }
            int token = -1;
            gather(rank == 0 ? (u64)(uint32_t)sh.found : 0ull, [&](uint32_t r, u64 x) { token = r == 0 ? (int)(uint32_t)x : token; });
            if (token >= 0) return done(token);
        } else {
            if (use_k) {
                auto one = [](uint32_t k, uint32_t) { return k ? 1ull : 0ull; };
                if (n_k <= LIST) {
                    to_list(bk, bk);
                    cut_list(k_left, one, [](uint32_t) { return 1ull; });
                } else {
                    cut_row(kk, one, [](uint32_t) { return 1ull; });
                }
            }
            if (p < 1.0f) {
                auto f = [&](uint32_t k, uint32_t j) { return stays(k, j) ? weigh(k) : 0ull; };
                u64 above = 0;
                if (use_k) W = over(f);
                const double t = ceil((double)fmaxf(p, 0.0f) * (double)W);
                const u64 want = t < 1.0 ? 1ull : (u64)t;
                bool in_list = !use_k && n_p <= LIST;
                if (in_list) {
                    to_list(p0, p1);
                    above = over([&](uint32_t k, uint32_t j) { return k && bin_of(k) < p0 ? f(k, j) : 0ull; });
                    const u64 inside = over([&](uint32_t k, uint32_t j) {
                        if (!k) return 0ull;
                        const int b = bin_of(k);
                        return b >= p0 && b <= p1 ? f(k, j) : 0ull;
                    });
                    in_list = above < want && want <= above + inside;
                }
                if (in_list) cut_list(want - above, f, [&](uint32_t k) { return weigh(k); });
                else cut_row(want, f, [&](uint32_t k) { return weigh(k); });
            }
            goto draw;
        }
        // the candidates did not hold top-p's cut: over the row
        {
            if (use_k) cut_row(kk, [](uint32_t k, uint32_t) { return k ? 1ull : 0ull; }, [](uint32_t) { return 1ull; });
            auto f = [&](uint32_t k, uint32_t j) { return stays(k, j) ? weigh(k) : 0ull; };
            if (use_k) W = over(f);
            const double t = ceil((double)fmaxf(p, 0.0f) * (double)W);
            cut_row(t < 1.0 ? 1ull : (u64)t, f, [&](uint32_t k) { return weigh(k); });
        }
    }
draw:
    // the draw: each warp sums a run of consecutive entries
    auto kept = [&](int i) -> u64 {
        const uint32_t k = i < n ? keys[i] : 0u;
        if (!k || !stays(k, (uint32_t)(base + i))) return 0;
        const double w = weigh.real(k);
        return w < mp_units ? 0ull : Weigh::whole(w);
    };
    const int run_len = ((a.slice + WARPS - 1) / WARPS + 31) / 32 * 32, i0 = warp * run_len, i1 = min(i0 + run_len, n);
    u64 mine = 0;
    for (int i = i0 + lane; i < i1; i += 32) mine += kept(i);
    mine = warp_sum(mine);
    __syncthreads();
    if (lane == 0) sh.warp[0][warp] = mine;
    if (tid == 0) sh.found = -1;
    __syncthreads();
    u64 before = 0, all = 0;
    for (int k = 0; k < WARPS; ++k) {
        if (k < warp) before += sh.warp[0][k];
        all += sh.warp[0][k];
    }
    u64 K = 0, front = 0;
    gather(all, [&](uint32_t r, u64 x) {
        if (r < rank) front += x;
        K += x;
    });
    const double uu = u_in > 0.0f ? (double)u_in : 0.0;
    u64 t = uu >= 1.0 ? K - 1 : (u64)(uu * (double)K);
    if (t > K - 1) t = K - 1;
    before += front;
    if (before <= t && t < before + mine) {  // this warp's run holds it
        for (int i = i0; i < i1; i += 32) {
            u64 x = kept(i + lane < i1 ? i + lane : n);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const u64 y = __shfl_up_sync(~0u, x, d);
                if (lane >= d) x += y;
            }
            const uint32_t hit = __ballot_sync(~0u, t < before + x);
            if (hit) {
                if (lane == 0) a.out[row] = base + i + __ffs(hit) - 1;
                break;
            }
            before += __shfl_sync(~0u, x, 31);
        }
    }
    cluster_sync();
}

template <typename T>
cudaError_t launch(const SampleArgs &in, cudaStream_t s) {
    SampleArgs a = in;
    // The smallest cluster whose slices stay below 16384 entries, so that two CTAs fit an SM; more CTAs where few rows
    // would leave SMs idle.
    int C = 1;
    while (C < 8 && ((a.vocab + C - 1) / C > 16384 || ((int64_t)a.n_rows * C * 2 <= dev::sm_count() && a.vocab / C > 4096))) C *= 2;
    a.slice = ((a.vocab + C - 1) / C + 7) / 8 * 8;
    const size_t smem = sizeof(Shared) + (size_t)a.slice * 4;
    cudaError_t e = dev::smem(sample_logits_kernel<T>, smem);
    if (e != cudaSuccess) return e;
    return launch_pdl_cluster(sample_logits_kernel<T>, dim3((unsigned)a.n_rows * C), dim3(THREADS), smem, s, dim3(C), a);
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
    if (n_rows > 1 << 24) return fail(ctx, KG_ERR_UNSUPPORTED, "sample: at most 16777216 rows");
    if (n_rows > 1 && ld < vocab) return fail(ctx, KG_ERR_INVALID_ARG, "sample: rows overlap (ld < vocab)");
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == KG_DT_F32 ? 4 : 2))
        return fail(ctx, KG_ERR_INVALID_ARG, "sample: logits not aligned to their type");
    if (!ctx) return fail(ctx, KG_ERR_INVALID_ARG, "null context");
    if (n_rows == 0) return KG_OK;
    DeviceGuard dg(ctx->device);
    if (dg.err != cudaSuccess) return cuda_fail(ctx, dg.err, "kg_sample_logits_dev");
    SampleArgs a{logits, n_rows > 1 ? ld : 0, n_rows, vocab, 0, temperature, top_k, top_p, min_p, u, tokens_out};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == KG_DT_F32 ? launch<float>(a, s) : dtype == KG_DT_BF16 ? launch<__nv_bfloat16>(a, s) : launch<__half>(a, s);
    return e == cudaSuccess ? KG_OK : cuda_fail(ctx, e, "kg_sample_logits_dev");
}
