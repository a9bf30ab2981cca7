// kg_pool_attn.cuh — what the two kernels of kg_pool_attend_dev share: their
// arguments, the walk over a CTA's part of the line of units, and the partial
// results that the joining kernel reads.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kg_async.cuh"
#include "kg_pool_ring.h"
#include "kg_serve.h"

namespace kg {
namespace serve {

constexpr int kBoxRows = 64;  // page rows of a TMA box at most
constexpr int kMaxParts = 320, kMaxLongParts = 160;  // CTAs of the two kernels' lines at most (2 and 1 on each of a B200's 148 SMs)

struct AttendArgs {
    Shape s;
    int n_req, total_q, width, page_size, n_pages;
    const int32_t *cu, *kv, *table;
    const void *q;
    void *out;
    int64_t q_row, q_head, o_row, o_head;
    float scale;  // times log2(e)
    int *err;
    int quick;  // clock cycles of the QUICK kernels' waits; 0: the usual kernels
    // partial results: slot 2 c of CTA c for the item its part begins inside, slot 2 c + 1 for the one it
    // ends inside without having begun in; `rows` rows of head_dim sums, then rows of (max, sum)
    float *part;
    int64_t slot_floats;
    int rows;
    int4 *meta;  // per slot: {0 unused, 1 used, 3 used and the item's end, request, head, tile}
};

// Probabilities are 2^(s - m), m a number near the row's maximum that all parts of the row count from (their sums and
// products scale alike). In bf16, which has f32's exponents, m is the maximum, or one that lags behind it by LAG at most.
// f16 has few exponents below 1: what is 2^-14 of the largest would lose bits and what is 2^-25 of it would be 0, while the
// row's sum holds it in full (a far maximum whose value is small, and a long flat rest: the rest was lost). There m lies UP
// below the maximum, or UP_LONG where it may lag, so that a probability reaches 2^15, the last power that f16 holds, and
// all bits are kept down to 2^-29 and 2^-26 of the largest. (LAG 2, 3, 4 and 8, a chunk of 2048 tokens over 18000 in f16:
// 544, 530, 519 and 507 us.)
template <typename T>
struct Cvt;
template <>
struct Cvt<__nv_bfloat16> {
    static constexpr float LAG = 8.0f, UP = 0.0f, UP_LONG = 0.0f;  // (LAG: of the long requests' kernel)
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <>
struct Cvt<__half> {
    static constexpr float LAG = 3.0f, UP = 15.0f, UP_LONG = UP - LAG;
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};

// m of a maximum; from 2^24 on f32 may have no number near enough to it, and no probability may leave f16's range
__device__ __forceinline__ float base_of(float top, float up) {
    if (up == 0.0f) return top;
    const float m = top - up;
    return top - m > up + 0.5f ? top : m;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The kernels are built twice: QUICK ones, for a test, whose waits run out after a.quick clock cycles (mbarrier.try_wait may
// sleep for longer, test_wait does not). Choosing at run time cost the long requests' kernel 6%.
template <bool QUICK>
__device__ __forceinline__ bool bounded_wait(uint64_t *bar, int parity, volatile int *abort_flag, const AttendArgs &a) {
    if (!QUICK) return as::mbar_wait(bar, parity, abort_flag, a.err);
    const long long t0 = clock64();
    do {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok)
                     : "r"(as::sa(bar)), "r"(parity)
                     : "memory");
        if (ok) return true;
    } while (!*abort_flag && clock64() - t0 < a.quick);
    *abort_flag = 1;
    atomicExch(a.err, (int)KG_ERR_TIMEOUT);
    return false;
}
// for what ends whatever else happened (bounded all the same)
__device__ __forceinline__ void wait_done(uint64_t *bar, int parity) {
    const long long t0 = clock64();
    while (!as::mbar_try(bar, parity) && clock64() - t0 < (1ll << 28)) {
    }
}
// The barriers of a ring of stages (kg_pool_ring.h), `bytes` in each.
template <bool QUICK>
struct Ring {
    uint64_t *full, *empty;
    uint32_t bytes;
    volatile int *abort_flag;
    const AttendArgs &a;
    __device__ __forceinline__ bool wait_full(int s, int parity) { return bounded_wait<QUICK>(&full[s], parity, abort_flag, a); }
    __device__ __forceinline__ bool wait_empty(int s, int parity) { return bounded_wait<QUICK>(&empty[s], parity, abort_flag, a); }
    __device__ __forceinline__ void arm(int s) { as::mbar_expect_tx(&full[s], bytes); }
    __device__ __forceinline__ void free(int s) { as::mbar_arrive(&empty[s]); }
    __device__ __forceinline__ bool all(bool x) { return __all_sync(~0u, x) != 0; }
    __device__ __forceinline__ void landed(int s, int parity) { wait_done(&full[s], parity); }
};

// Shared-memory form of K and V: groups of 8 positions, each [head_dim / 64][8
// rows][128 bytes] with the 128-byte swizzle. One TMA box brings all of a page's
// rows of one head (64 at most) in this order: the pool is mapped as
//   [64 elements][8 rows][head_dim / 64][row groups][page and head]
// where the last axis counts in steps of `unit` elements, the greatest common
// divisor of the page and head strides. (A box for every 64 elements of a 16-row
// page, 2 KB each, kept the loads of a prompt chunk behind its products.)
struct PoolMap {
    CUtensorMap k, v;
    int page_step, head_step, outside;  // in the last axis; `outside` lies behind it: such a box becomes zeros
};
template <int D>
__device__ __forceinline__ uint32_t kv_offset(int row, int chunk) {  // of a 16-byte chunk, before the swizzle
    return (row >> 3) * (D * 16) + (chunk >> 3) * 1024 + (row & 7) * 128 + (chunk & 7) * 16;
}
__device__ __forceinline__ void tma_load_5d(void *dst, const CUtensorMap *tm, int row_group, int place, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3, %4}], "
        "[%5];\n" ::"r"(as::sa(dst)),
        "l"(tm), "r"(0), "r"(row_group), "r"(place), "r"(as::sa(bar))
        : "memory");
}

// the map itself into the loader's cache, before its first use
__device__ __forceinline__ void prefetch_map(const CUtensorMap *tm) { asm volatile("prefetch.tensormap [%0];" ::"l"(tm) : "memory"); }

// 4-D tiled load: the rows of q of one K/V head, 64 elements wide
__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *tm, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];\n" ::"r"(as::sa(dst)),
        "l"(tm), "r"(x), "r"(y), "r"(z), "r"(w), "r"(as::sa(bar))
        : "memory");
}

// lengths of request r, zeros where they cannot be used
__device__ __forceinline__ bool req_len(const AttendArgs &a, int r, int &q0, int &q, int &kv) {
    q0 = a.cu[r];
    const int q1 = a.cu[r + 1];
    kv = a.kv[r];
    const bool ok = lengths_ok(q0, q1, kv, a.total_q, min((int64_t)a.width * a.page_size, (int64_t)kMaxKv));
    q = ok ? q1 - q0 : 0;
    if (!ok) kv = 0;
    return ok;
}

// This CTA's part (of parts_of() ones): where it begins and how many units it has.
// Every thread of the block calls it (NT threads); `sm` holds 2 NT / 32 + 2 numbers.
template <int NT, bool LONG>
__device__ void find_part(const AttendArgs &a, int c, int parts, int least, long long *sm, int &req, long long &off,
                          long long &units) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.n_req + NT - 1) / NT, r0 = min(tid * per, a.n_req), r1 = min(r0 + per, a.n_req);
    long long mine = 0, items = 0;
    for (int r = r0; r < r1; ++r) {
        int q0, q, kv;
        if (!req_len(a, r, q0, q, kv) && c == 0) reject(a.err);
        mine += request_units(a.s, LONG, q, kv);
        items += request_items(a.s, LONG, q, kv);
    }
    long long incl = mine;
    for (int d = 1; d < 32; d <<= 1) {
        const long long u = __shfl_up_sync(~0u, incl, d);
        if (lane >= d) incl += u;
    }
    const int few = __reduce_add_sync(~0u, (int)min(items, 65536ll));  // enough to compare with the CTAs there are
    if (lane == 31) {
        sm[warp] = incl;
        sm[NT / 32 + warp] = few;
    }
    __syncthreads();
    long long before = incl - mine, total = 0;
    items = 0;
    for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) before += sm[w];
        total += sm[w];
        items += sm[NT / 32 + w];
    }
    parts = parts_of(total, items, parts, least);
    const long long b = c < parts ? part_begin(total, c, parts) : 0, e = c < parts ? part_begin(total, c + 1, parts) : 0;
    units = e - b;
    if (units > 0 && before <= b && b < before + mine) {
        long long at = before;
        for (int r = r0; r < r1; ++r) {
            int q0, q, kv;
            req_len(a, r, q0, q, kv);
            const long long n = request_units(a.s, LONG, q, kv);
            if (b < at + n) {
                sm[2 * (NT / 32)] = r;
                sm[2 * (NT / 32) + 1] = b - at;
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    req = units > 0 ? (int)sm[2 * (NT / 32)] : 0;
    off = units > 0 ? sm[2 * (NT / 32) + 1] : 0;
}

// The items of a part, in order.
template <bool LONG>
struct Walk {
    int r, q0, q, kv;
    Place p;
    int n;           // units of the item here
    long long left;  // units after it
    __device__ __forceinline__ void start(const AttendArgs &a, int req, long long off, long long units) {
        r = req;
        left = units;
        if (units <= 0) return;
        req_len(a, r, q0, q, kv);
        p = place_of(a.s, LONG, q, kv, off);
        take();
    }
    __device__ __forceinline__ void take() {
        n = (int)min(left, (long long)(p.units - p.unit));
        left -= n;
    }
    // to the next item; false at the end
    __device__ __forceinline__ bool next(const AttendArgs &a) {
        if (left <= 0) return false;
        p.unit = 0;
        if (LONG && p.tile + 1 < long_tiles(a.s, q)) {
            ++p.tile;
        } else {
            p.tile = 0;
            if (++p.head == a.s.n_kv) {
                p.head = 0;
                do {
                    ++r;
                    req_len(a, r, q0, q, kv);
                } while (request_units(a.s, LONG, q, kv) == 0);
            }
        }
        p.units = LONG ? long_units(a.s, q, kv, p.tile) : short_units(a.s, q, kv);
        take();
        return true;
    }
    __device__ __forceinline__ bool whole() const { return p.unit == 0 && n == p.units; }
    // slot of a partial item: 0 when its first units are another CTA's
    __device__ __forceinline__ int slot() const { return p.unit == 0 ? 1 : 0; }
    __device__ __forceinline__ bool ends() const { return p.unit + n == p.units; }
};

// The long requests' kernel (kg_pool_long.cu), `parts` CTAs.
cudaError_t attend_long(const PoolMap &kv, const AttendArgs &a, bool bf16, int head_dim, int parts, cudaStream_t s);

}  // namespace serve
}  // namespace kg
