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
// global memory once. A histogram of (max - x) / T, of entries (in steps of 1/64) or,
// for top-p, of entries and weights (in steps of 1/64 of an octave of w), says in which
// step each cut lies (each CTA adds up its share of the steps):
//   - where the candidates down to that step are at most 2048 (small top-k, a peaked
//     row), they go to the cluster's first CTA, which sorts them and finishes the row
//     alone;
//   - else the entries of that one step, at most 4096, go there and are sorted, the cut
//     is where the running sum from what lies above them arrives; the token is drawn by
//     all CTAs;
//   - where a step holds more (rows of equal values), by bisection over the whole row.
// Bound by the latency of a row's steps (64 rows of 32000 in 44 us; 21 us where every
// token stays) and by the weights: 256 nucleus rows of 131072 in 500 us, 33 clusters at a
// time in eight rounds (read alone, 10 us). A weight costs about 14 operations in 64 bits,
// at half the 32-bit rate, and is computed once for top-p's histogram and once for what
// is drawn from; 64 registers a thread for two CTAs on an SM spill 124 bytes.
// Sorting up to 4096 entries of a step, against 2048 and the bisection before it, and
// candidates in the first CTA: 256 x 131072 nucleus rows of normal logits take 8% to 12%
// longer at a deviation of 0.5 to 4 (bf16, 2: 460 -> 500 us), but 620 us in place of 1500
// at 0.3, where steps are crowded, and 690 in place of 2360 at 0.2; 64 mixed rows of 32000
// 57 -> 49 us, 285 -> 79 at 0.05.
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

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 2048, LIST = 2048, STEP_LIST = 2 * LIST;
constexpr int PER = LIST / THREADS;  // candidates of a thread

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
__device__ __forceinline__ int bits_of(u64 v, int at, int bits) { return (int)(v >> at & ((1ull << bits) - 1)); }
__device__ __forceinline__ u64 remote_u64(uint32_t a) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void remote_store(uint32_t a, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }

struct alignas(16) Shared {
    double tab[64];      // 2^(j / 64)
    u64 warp[2][WARPS];  // block sums
    u64 red[2][3];       // this CTA's part of what a cluster shares
    u64 cut;             // an entry of `sorted`
    uint32_t range[2];   // keys of a step
    uint32_t queue[WARPS][64];
    union {
        struct {
            uint32_t count[BINS], low[BINS], high[BINS];  // entries and weights (two words) of this CTA's slice by step
        };
        struct {
            u64 list[LIST];    // key << 32 | index, by index, of the first CTA
            u64 sorted[LIST];  // key << 32 | ~index, the largest first (a step's entries: from `list` on)
        };
    };
};

static_assert(sizeof(Shared) % 16 == 0, "the keys behind it are read 16 bytes at a time");

// The weight's arithmetic: 2^y by a table of 2^(j / 64) and the series of 2^r, |r| <= 1/128 (the first term left out is
// below 2^-54). -64 y to the nearest integer is also the entry's step of the histogram. No branches: several run at a time.
struct Weigh {
    double c, xmax;  // log2(e) / T
    uint32_t kmax;
    bool inf;
    const double *tab;
    __device__ __forceinline__ double real(uint32_t k) const {  // in units
        int step;
        return real(k, step);
    }
    __device__ __forceinline__ double real(uint32_t k, int &step) const {
        if (inf) {  // (of the whole row)
            step = k == kmax ? 0 : BINS - 1;
            return k == kmax ? 17592186044416.0 : 0.0;
        }
        const double y = fmax(((double)value_of(k) - xmax) * c, -47.0);  // 2^-47 counts as 0; so does key 0, NaN
        const double t = fma(y, 64.0, 6755399441055744.0);  // rounds to an integer in the low bits
        const int n = __double2loint(t);
        const double r = fma(t - 6755399441055744.0, -0.015625, y);
        double p = 0.00133335581464284411;  // ln(2)^n / n!
        p = fma(p, r, 0.00961812910762847688);
        p = fma(p, r, 0.0555041086648215762);
        p = fma(p, r, 0.240226506959100694);
        p = fma(p, r, 0.693147180559945286);
        p = fma(p, r, 1.0);
        p *= tab[n & 63];
        step = min(-n, BINS - 1);
        return __hiloint2double(__double2hiint(p) + (((n >> 6) + 44) << 20), __double2loint(p));
    }
    static __device__ __forceinline__ u64 whole(double w) {  // w below 2^51, to the nearest
        return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 operator()(uint32_t k) const { return whole(real(k)); }
};

// Values of 16 bits leave the low bits of their keys alike: a bisection over keys need not look at them.
template <typename T>
struct Spare;
template <>
struct Spare<float> {
    static constexpr int bits = 0;
};
template <>
struct Spare<__half> {
    static constexpr int bits = 13;
};
template <>
struct Spare<__nv_bfloat16> {
    static constexpr int bits = 16;
};
template <typename T>
__device__ __forceinline__ uint32_t key_at(uint32_t q) {  // the key whose upper bits are q
    constexpr int b = Spare<T>::bits;
    const uint32_t k = q << b;
    return k & 0x80000000u ? k : k | ((1u << b) - 1u);
}

// sum over the warp, below 2^63: three parts of 26 bits whose sums stay in 32
__device__ __forceinline__ u64 warp_sum(u64 v) {
    const uint32_t a = __reduce_add_sync(~0u, (uint32_t)v & 0x3ffffffu), b = __reduce_add_sync(~0u, (uint32_t)(v >> 26) & 0x3ffffffu),
                   c = __reduce_add_sync(~0u, (uint32_t)(v >> 52));
    return (u64)a + ((u64)b << 26) + ((u64)c << 52);
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
    auto scan = [&](u64 v) {  // exclusive, over the block's threads
        u64 x = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const u64 y = __shfl_up_sync(~0u, x, d);
            if (lane >= d) x += y;
        }
        u64 *to = sh.warp[flip & 1];
        ++flip;
        if (lane == 31) to[warp] = x;
        __syncthreads();
        u64 before = 0;
        for (int k = 0; k < warp; ++k) before += to[k];
        return before + x - v;
    };
    int turn = 0;
    // every CTA's values (v, x, y: the same in all its threads, or those of the thread that names them by `mine`): f(rank, v, x, y)
    auto share = [&](bool mine, u64 v, u64 x, u64 y, auto f) {
        u64 *to = sh.red[turn & 1];
        if (mine) {
            to[0] = v;
            to[1] = x;
            to[2] = y;
        }
        __syncwarp();
        cluster_sync();
        u64 got[8][3];
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r)
            if (r < C) {
                const uint32_t at = remote(to, r);
                got[r][0] = remote_u64(at);
                got[r][1] = remote_u64(at + 8);
                got[r][2] = remote_u64(at + 16);
            }
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r)
            if (r < C) f(r, got[r][0], got[r][1], got[r][2]);
        ++turn;
    };
    auto gather = [&](u64 v, auto f) {
        u64 *to = sh.red[turn & 1];
        if (tid == 0) to[0] = v;
        __syncwarp();
        cluster_sync();
        u64 got[8];
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r)
            if (r < C) got[r] = remote_u64(remote(to, r));
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r)
            if (r < C) f(r, got[r]);
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
    if (tid < 4 && n + tid < (n + 3) / 4 * 4) keys[n + tid] = 0;  // read four at a time
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
    const bool has_p = p < 1.0f;
    // an entry's step; never falls as the key falls
    auto bin_of = [&](uint32_t k) {
        if (has_p) {
            int b;
            weigh.real(k, b);
            return b;
        }
        return k == kmax ? 0 : min(BINS - 1, (int)((xmax - value_of(k)) * step));
    };

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
        constexpr int sp = Spare<T>::bits;
        uint32_t c = 0;
        for (uint32_t bit = 0x80000000u >> sp; bit; bit >>= 1) {
            const uint32_t t = c | bit;
            if (over([&](uint32_t k, uint32_t j) { return k >> sp >= t ? f(k, j) : 0ull; }) >= want) c = t;
        }
        c = key_at<T>(c);
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
    auto pick = [&](u64 K) {  // the place in the running sum that the given number names
        const double uu = u_in > 0.0f ? (double)u_in : 0.0;
        const u64 t = uu >= 1.0 ? K - 1 : (u64)(uu * (double)K);
        return t > K - 1 ? K - 1 : t;
    };
    auto part_of = [&](u64 W) {  // what top-p has to reach
        const double t = ceil((double)fmaxf(p, 0.0f) * (double)W);
        return t < 1.0 ? 1ull : (u64)t;
    };

    // each warp looks after a run of consecutive entries of the slice
    const int run_len = ((a.slice + WARPS - 1) / WARPS + 31) / 32 * 32, i0 = warp * run_len, i1 = min(i0 + run_len, n);
    // The first CTA's list (m_list entries in the order of the indexes), sorted by key and index: in the first CTA only. A
    // pair's places lie in its warp's 64 where the stride is at most 32.
    int m_list = 0;
    u64 *sorted = nullptr;
    auto sort_list = [&](bool in_place) {
        sorted = in_place ? sh.list : sh.sorted;
        int N = 64;
        while (N < m_list) N <<= 1;
        for (int i = tid; i < N; i += THREADS) sorted[i] = i < m_list ? sh.list[i] ^ 0xffffffffull : 0ull;
        __syncthreads();
        for (int size = 2; size <= N; size <<= 1)
            for (int stride = size / 2; stride; stride >>= 1) {
                for (int q = tid; q < N / 2; q += THREADS) {
                    const int i = 2 * q - (q & (stride - 1)), j = i + stride;
                    const u64 x = sorted[i], y = sorted[j];
                    if ((x < y) == ((i & size) == 0)) {
                        sorted[i] = y;
                        sorted[j] = x;
                    }
                }
                if (stride > 32 || (stride == 1 && size >= 64)) __syncthreads();
                else __syncwarp();
            }
    };
    auto cut_at = [&](u64 e) {  // behind entry e
        ck = (uint32_t)(e >> 32);
        ci = (uint32_t)~e + 1;
    };
    // the cut behind the first of the leading `count` sorted entries at which the sum of weights reaches part_of(W) - above
    // (W: theirs, where `own`, of at most LIST)
    auto cut_weights = [&](int count, bool own, u64 W, u64 above) {
        for (int first = 0; first < count; first += LIST) {
            u64 v[PER], here = 0;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int i = first + tid * PER + e;
                v[e] = i < count ? weigh((uint32_t)(sorted[i] >> 32)) : 0ull;
                here += v[e];
            }
            u64 run = scan(here);
            const u64 all = block_sum(here);
            if (own) W = all;
            const u64 want = part_of(W) - above;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                if (run < want && want <= run + v[e]) sh.cut = sorted[first + tid * PER + e];
                run += v[e];
            }
            if (want <= all) break;
            above += all;
        }
        __syncthreads();
        cut_at(sh.cut);
    };
    // the first CTA's cut, for every CTA
    auto share_cut = [&]() {
        u64 x = 0;
        gather((u64)ck << 32 | ci, [&](uint32_t r, u64 v) { x = r == 0 ? v : x; });
        ck = (uint32_t)(x >> 32);
        ci = (uint32_t)x;
    };
    // The smallest key whose step is at most b (32 tries at a time; the first warp).
    auto smallest_key = [&](int b) {
        uint32_t lo = 0x00800000u, hi = kmax;  // the answer is in [lo, hi]; lo is the key of the lowest finite value
        while (lo < hi) {
            const uint32_t span = (hi - lo) / 32 + 1, t = lo + lane * span < hi && lo + lane * span >= lo ? lo + lane * span : hi;
            const uint32_t yes = __ballot_sync(~0u, bin_of(t) <= b);  // from some lane on
            const int l = __ffs(yes) - 1;                            // (the last lane's key may be hi itself, whose step is)
            const uint32_t at = yes ? __shfl_sync(~0u, t, l) : hi, under = yes && l == 0 ? lo : __shfl_sync(~0u, t, yes ? l - 1 : 31) + 1;
            lo = yes && l == 0 ? at : under;
            hi = at;
        }
        return hi;
    };
    // live entries whose bin is in [b0, b1] and that stay, into the first CTA's list
    auto to_list = [&](int b0, int b1) {
        if (warp == 0) {
            const uint32_t lo = smallest_key(b1), over = b0 > 0 ? smallest_key(b0 - 1) : 0u;
            if (lane == 0) {
                sh.range[0] = lo;
                sh.range[1] = b0 > 0 ? over - 1 : kmax;
            }
        }
        __syncthreads();
        const uint32_t k_lo = sh.range[0], k_hi = sh.range[1];
        const bool whole = ck == 1;  // no cut so far
        u64 in = 0;  // of this thread's entries of the warp's run
        uint32_t found = 0;
        for (int i = i0, e = 0; i < i1; i += 32, ++e) {
            const uint32_t k = i + lane < i1 ? keys[i + lane] : 0u;
            const bool yes = k >= k_lo && k <= k_hi && (whole || stays(k, (uint32_t)(base + i + lane)));
            found += __popc(__ballot_sync(~0u, yes));
            if (yes) in |= 1ull << e;
        }
        u64 *w = sh.warp[flip & 1];
        ++flip;
        if (lane == 0) w[warp] = found;
        __syncthreads();
        uint32_t at = 0, all = 0;
        for (int k = 0; k < WARPS; ++k) {
            if (k < warp) at += (uint32_t)w[k];
            all += (uint32_t)w[k];
        }
        m_list = 0;
        gather(all, [&](uint32_t r, u64 x) {  // (the histograms, which lie under the list, have been read)
            if (r < rank) at += (uint32_t)x;
            m_list += (int)x;
        });
        const uint32_t dst = remote(sh.list, 0);
        for (int i = i0, e = 0; i < i1; i += 32, ++e) {
            const bool yes = in >> e & 1;
            const uint32_t who = __ballot_sync(~0u, yes);
            const uint32_t to = at + __popc(who & ((1u << lane) - 1));
            if (yes && to < STEP_LIST) remote_store(dst + to * 8, (u64)keys[i + lane] << 32 | (uint32_t)(base + i + lane));
            at += __popc(who);
        }
        __syncwarp();
        cluster_sync();
    };

    const u64 kk = want_k > 0 && want_k < a.vocab ? (u64)want_k : 0ull;
    if (kk || has_p) {
        for (int i = tid; i < BINS; i += THREADS) sh.count[i] = sh.low[i] = sh.high[i] = 0;
        __syncthreads();
        for (int i = tid * 4; i < n; i += THREADS * 4) {
            const uint4 k4 = *reinterpret_cast<const uint4 *>(keys + i);
            const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
            int b[4];
            u64 w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (has_p) {
                    w[e] = Weigh::whole(weigh.real(k[e], b[e]));
                } else {
                    b[e] = bin_of(k[e]);
                    w[e] = 0ull;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (k[e] == 0) continue;
                atomicAdd(&sh.count[b[e]], 1u);
                const uint32_t lo = (uint32_t)w[e];
                uint32_t hi = (uint32_t)(w[e] >> 32);
                if (lo && atomicAdd(&sh.low[b[e]], lo) > ~lo) ++hi;
                if (hi) atomicAdd(&sh.high[b[e]], hi);
            }
        }
        __syncwarp();
        cluster_sync();
        // this CTA's share of the steps: entries and weights of the whole row
        const int share_bins = BINS / (int)C, nb = max(1, share_bins / THREADS);
        const bool owner = tid * nb < share_bins;
        const int first = (int)rank * share_bins + tid * nb;
        u64 c[4], w[4], c_all = 0, w_all = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            c[j] = w[j] = 0;
            if (owner && j < nb) {
                uint32_t x[8], y[8], z[8];
                const int b = first + j;
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r)
                    if (r < C) {
                        x[r] = remote_u32(remote(&sh.count[b], r));
                        y[r] = has_p ? remote_u32(remote(&sh.low[b], r)) : 0u;
                        z[r] = has_p ? remote_u32(remote(&sh.high[b], r)) : 0u;
                    }
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r)
                    if (r < C) {
                        c[j] += x[r];
                        w[j] += ((u64)z[r] << 32) + y[r];
                    }
            }
            c_all += c[j];
            w_all += w[j];
        }
        u64 c_run = scan(c_all), w_run = has_p ? scan(w_all) : 0ull, live = 0, W = 0;
        share(tid == THREADS - 1, c_run + c_all, w_run + w_all, 0, [&](uint32_t r, u64 x, u64 y, u64) {
            if (r == rank) {
                c_run += live;
                w_run += W;
            }
            live += x;
            W += y;
        });
        // The step that holds the k-th entry: {step, entries before it, entries in it}, 12, 20 and 20 bits and a mark.
        auto packed = [&](int b, u64 before, u64 in) { return 1ull << 63 | (u64)b << 40 | before << 20 | in; };
        const bool use_k = kk && kk < live;
        int bk = BINS, before_k = 0, n_k = 0;
        if (use_k) {
            u64 x = c_run, hit = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (owner && x < kk && kk <= x + c[j]) hit = packed(first + j, x, c[j]);
                x += c[j];
            }
            if (tid == 0) sh.red[turn & 1][0] = 0;
            __syncthreads();
            u64 got = 0;
            share(hit != 0, hit, 0, 0, [&](uint32_t, u64 v, u64, u64) { got = max(got, v); });
            bk = bits_of(got, 40, 12);
            before_k = bits_of(got, 20, 20);
            n_k = bits_of(got, 0, 20);
        }
        // The step that holds the place where the weights reach `want` (among the first bk, or bk itself).
        u64 above = 0;
        int bp = BINS, before_p = 0, n_p = 0;
        auto find_weight = [&](u64 want) {
            u64 x = w_run, y = c_run, hit = 0, hit_above = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = first + j;
                if (owner && j < nb && x < want && (b < bk ? want <= x + w[j] : b == bk)) {
                    hit = packed(b, y, c[j]);
                    hit_above = x;
                }
                x += w[j];
                y += c[j];
            }
            if (tid == 0) sh.red[turn & 1][0] = 0;
            __syncthreads();
            u64 got = 0;
            share(hit != 0, hit, hit_above, 0, [&](uint32_t, u64 v, u64 ab, u64) {
                if (v) {
                    got = v;
                    above = ab;
                }
            });
            bp = bits_of(got, 40, 12);
            before_p = bits_of(got, 20, 20);
            n_p = bits_of(got, 0, 20);
        };
        if (!use_k && has_p) find_weight(part_of(W));
        const int all_of = use_k ? before_k + n_k : before_p + n_p;
        if ((use_k || has_p) && all_of <= LIST) {
            // Few candidates: the first CTA finishes the row.
            to_list(0, use_k ? bk : bp);
            if (rank == 0) {
                sort_list(false);
                if (use_k) cut_at(sorted[kk - 1]);
                if (has_p) cut_weights(use_k ? (int)kk : m_list, use_k, W, 0);
                u64 v[PER], here = 0;
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int i = tid * PER + e;
                    const u64 x = i < m_list ? sh.list[i] : 0ull;
                    const uint32_t k = (uint32_t)(x >> 32);
                    const double w = weigh.real(k);
                    v[e] = k && stays(k, (uint32_t)x) && w >= mp_units ? Weigh::whole(w) : 0ull;
                    here += v[e];
                }
                u64 run = scan(here);
                const u64 t = pick(block_sum(here));
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    if (run <= t && t < run + v[e]) a.out[row] = (int)(uint32_t)sh.list[tid * PER + e];
                    run += v[e];
                }
            }
            return;  // (the others' shared memory is not read any more)
        }
        if (use_k) {
            if (n_k <= STEP_LIST) {
                to_list(bk, bk);
                if (rank == 0) {
                    sort_list(true);
                    cut_at(sorted[kk - before_k - 1]);
                }
                share_cut();
            } else {
                cut_row(kk, [](uint32_t k, uint32_t) { return k ? 1ull : 0ull; }, [](uint32_t) { return 1ull; });
            }
        }
        if (has_p) {
            auto f = [&](uint32_t k, uint32_t j) { return stays(k, j) ? weigh(k) : 0ull; };
            if (use_k) {
                W = over(f);
                find_weight(part_of(W));
            }
            const u64 want = part_of(W);
            if (n_p <= STEP_LIST) {
                to_list(bp, bp);
                if (rank == 0) {
                    sort_list(true);
                    cut_weights(m_list, false, W, above);
                }
                share_cut();
            } else {
                cut_row(want, f, [&](uint32_t k) { return weigh(k); });
            }
        }
    }
    // the draw: each warp sums a run of consecutive entries
    auto kept = [&](uint32_t k) -> u64 {  // of a key that stays
        const double w = weigh.real(k);
        return k == 0 || w < mp_units ? 0ull : Weigh::whole(w);
    };
    u64 mine = 0;
    if (ck == 1) {  // no cut
        for (int i = i0 + lane; i < i1; i += 32) mine += kept(keys[i]);
    } else {  // what stays is queued, so that weights are computed for 32 of them at a time
        uint32_t *queue = sh.queue[warp];
        int q = 0;
        for (int i = i0; i < i1; i += 32) {
            const uint32_t k = i + lane < i1 ? keys[i + lane] : 0u;
            const bool in = k && stays(k, (uint32_t)(base + i + lane));
            const uint32_t who = __ballot_sync(~0u, in);
            if (in) queue[q + __popc(who & ((1u << lane) - 1))] = k;
            q += __popc(who);
            __syncwarp();
            if (q >= 32) {
                mine += kept(queue[lane]);
                const uint32_t rest = queue[32 + lane];
                __syncwarp();
                queue[lane] = rest;
                q -= 32;
                __syncwarp();
            }
        }
        if (lane < q) mine += kept(queue[lane]);
    }
    mine = warp_sum(mine);
    __syncthreads();
    if (lane == 0) sh.warp[0][warp] = mine;
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
    const u64 t = pick(K);
    before += front;
    if (before <= t && t < before + mine) {  // this warp's run holds it
        for (int i = i0; i < i1; i += 32) {
            const uint32_t k = i + lane < i1 ? keys[i + lane] : 0u;
            u64 x = k && stays(k, (uint32_t)(base + i + lane)) ? kept(k) : 0ull;
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
    while (C < 8 && ((a.vocab + C - 1) / C > 16384 || ((int64_t)a.n_rows * C <= dev::sm_count() && a.vocab / C > 4096))) C *= 2;
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
