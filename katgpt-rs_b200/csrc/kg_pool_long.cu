// kg_pool_long.cu — the long requests of kg_pool_attend_dev (more than 64 rows
// per K/V head: prompt chunks) on tcgen05.
//
// An item is 2 x TQ tokens of one K/V head, TQ = floor(128 / group): two tiles of
// up to 128 rows (token, query head of the group), one row per tensor-memory lane.
// Per unit of 128 positions and tile t:
//   S_t = Q_t K^T      (M 128, N 128, both operands in shared memory)
//   P_t = 2^(S_t - m)  (a thread owns a row: its maximum and sum need no exchange)
//   O_t += P_t V       (M 128, N head_dim, P_t from tensor memory over S_t)
// Warps: 0 loads (TMA, a box per page), 1 issues the products, 2..5
// and 6..9 are the rows of tile 0 and tile 1. The products go P_0 V, Q_0 K^T, P_1 V,
// Q_1 K^T in turn from one thread, so that the tiles stay half a step apart: one tile's
// rows are exponentiated while the other tile's products run. (Two issuing threads let
// the tiles fall into step, both waiting for the tensor pipe and then both for the
// exponentials: 4640 cycles a pair of units at 1.70 GHz.)
// 2048 tokens over 18000 positions, 32 query and 8 K/V heads of 128, bf16: 497 us between
// pauses, 555 to 565 us back to back (1,010 to 1,030 TFLOP/s, under the power cap), f16 527;
// heads of 64 455 us and 466. A pair of units takes about 3,150 cycles, of which the products
// 2,055 and the exponentials 2,048 run beside each other: bound by the chain scores ->
// exponentials -> values -> next scores of one tile.
// A row's O is rescaled only when its maximum has grown by more than 2^LAG since the
// last time: 2^8 in bf16, whose P then reaches at most 2^8; 2^3 in f16, whose P has to
// use the range that it has (Cvt).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "kg_dev.cuh"
#include "kg_pdl.cuh"
#include "kg_pool_attn.cuh"
#include "kg_tc.cuh"

namespace kg {
namespace serve {
namespace {

using namespace as;

constexpr int LONG_THREADS = 320, LONG_LEAST = 2;

template <int D>
struct LongCfg {
    static constexpr int HALF = 128 * 128;           // 128 rows x 64 elements
    static constexpr int OP = HALF * (D / 64);       // a Q tile, or K or V of a unit
    static constexpr int SLOTS = D == 64 ? 6 : 4;    // K and V in turn
    static constexpr int BARS = 2 * SLOTS + 2 + 8 + 1;
    static constexpr int SMEM = 1024 + 2 * OP + SLOTS * OP + BARS * 8 + 16;
};

// 64 columns of this thread's lane, the wait inside
__device__ __forceinline__ void ld64w(uint32_t taddr, float (&v)[64]) {
    uint32_t r[64];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
// 16 columns, the wait inside
__device__ __forceinline__ void ld16w(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// one lane of a converged warp, always the same one (its products stay in order)
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred P;\n elect.sync _|P, 0xffffffff;\n selp.u32 %0, 1, 0, P;\n}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(~0u, x, 0); }

// two f32 at a time
__device__ __forceinline__ unsigned long long two(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void halves(unsigned long long v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

struct LongMaps {
    CUtensorMap q;
    PoolMap kv;
};

template <typename T, int D, bool QUICK>
__global__ void __launch_bounds__(LONG_THREADS, 1) attend_long_kernel(const __grid_constant__ LongMaps maps, const AttendArgs a) {
    using C = LongCfg<D>;
    extern __shared__ __align__(1024) uint8_t raw[];
    uint8_t *sm = raw + ((1024u - (sa(raw) & 1023u)) & 1023u);
    uint8_t *sq = sm, *slots = sm + 2 * C::OP;
    uint64_t *full = reinterpret_cast<uint64_t *>(slots + C::SLOTS * C::OP), *empty = full + C::SLOTS;
    uint64_t *qfull = empty + C::SLOTS, *qempty = qfull + 1;
    uint64_t *sfull = qempty + 1, *pvdone = sfull + 2, *pready = pvdone + 2;  // [2] by tile, pready [tile][half]
    uint64_t *last = pready + 4;
    uint32_t *tslot = reinterpret_cast<uint32_t *>(last + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tslot + 1);
    __shared__ long long part_sm[2 * (LONG_THREADS / 32) + 2];
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31, c = blockIdx.x;
    const int group = a.s.group, tq = a.s.tile / 2;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(qfull, 1);
        mbar_init(qempty, 1);
        mbar_init(last, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sfull[t], 1);
            mbar_init(&pready[2 * t], 4);
            mbar_init(&pready[2 * t + 1], 4);
            mbar_init(&pvdone[t], 1);
        }
        *abort_flag = 0;
        mbar_fence_init();
        prefetch_map(&maps.q);
        prefetch_map(&maps.kv.k);
        prefetch_map(&maps.kv.v);
    }
    pdl_wait();
    pdl_launch();  // the short requests' kernel may take the SMs that this one leaves free
    int req;
    long long off, units;
    find_part<LONG_THREADS, true>(a, c, gridDim.x, LONG_LEAST, part_sm, req, off, units);
    if (threadIdx.x < 2) a.meta[2 * c + threadIdx.x].x = 0;
    __syncthreads();
    if (units == 0) return;
    if (warp == 0) tc::alloc(tslot, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tb = *tslot;
    Walk<true> w;
    w.start(a, req, off, units);
    // units of tile t's rows within the item's run [unit, unit + n): the first n_of(t)
    auto n_of = [&](int t) {
        const int first = (w.p.tile * 2 + t) * tq;
        if (first >= w.q) return 0;
        const int lim = row_limit(a.s, w.q, w.kv, min(first + tq, w.q) - 1);
        const int u = lim > 0 ? (lim - 1) / kLongUnit + 1 : 0;
        return max(0, min(w.n, u - w.p.unit));
    };

    if (warp == 0) {  // loads: a ring of K and V in turn, and one of a single stage for the item's rows of q
        Ring<QUICK> ring{full, empty, C::OP, abort_flag, a}, q_ring{qfull, qempty, 0, abort_flag, a};
        const int rows = min(a.page_size, kBoxRows), pages = kLongUnit / rows;  // a box each
        int it = 0, item = 0;
        bool ok = true;
        do {
            if (lane == 0) {
                const int first = w.p.tile * 2 * tq, tiles = first + tq < w.q ? 2 : 1;
                q_ring.bytes = tiles * (D / 64) * tq * group * 128;
                ok = ring_claim(q_ring, 1, item);
                if (ok) {
                    for (int t = 0; t < tiles; ++t)
                        for (int h = 0; h < D / 64; ++h)
                            tma_load_4d(sq + t * C::OP + h * C::HALF, &maps.q, h * 64, 0, w.p.head, w.q0 + first + t * tq, qfull);
                }
            }
            ok = __shfl_sync(~0u, ok, 0);
            item += ok;
            for (int u = 0; ok && u < w.n; ++u) {
                const int pos = (w.p.unit + u) * kLongUnit + lane * rows;
                int place = maps.kv.outside;
                if (lane < pages && pos < w.kv) {
                    const int e = a.table[(int64_t)w.r * a.width + pos / a.page_size];
                    if (e >= 0 && e < a.n_pages) place = e * maps.kv.page_step + w.p.head * maps.kv.head_step;
                    else reject(a.err);
                }
                for (int kv = 0; kv < 2; ++kv, ++it) {
                    const int s = it % C::SLOTS;
                    if (lane == 0) ok = ring_claim(ring, C::SLOTS, it);
                    ok = __shfl_sync(~0u, ok, 0);
                    if (!ok) break;
                    if (lane < pages)
                        tma_load_5d(slots + s * C::OP + lane * rows * D * 2, kv ? &maps.kv.v : &maps.kv.k, pos % a.page_size / 8, place, &full[s]);
                }
            }
        } while (ok && w.next(a));
        ring_drain(q_ring, 1, item);
        ring_drain(ring, C::SLOTS, it);
    } else if (warp == 1) {  // products, tile 0 and tile 1 in turn
        // The whole warp walks the loop and one lane issues: descriptors then stay in uniform registers. From inside a
        // one-lane branch a product took about 110 cycles to issue, against 64 to run.
        {
            constexpr int FMT = std::is_same<T, __half>::value ? 0 : 1;
            constexpr uint32_t IDS = tc::idesc_f16(FMT, 128, 128), IDO = tc::idesc_f16(FMT, 128, D, 0, 1);
            int it = 0, item = 0, cnt[2] = {0, 0};
            bool ok = true;
            auto wait = [&](uint64_t *b, int parity) { return __all_sync(~0u, bounded_wait<QUICK>(b, parity, abort_flag, a)) != 0; };
            auto wait_slot = [&](int step) { return wait(&full[step % C::SLOTS], (step / C::SLOTS) & 1); };
            auto scores = [&](int t, int step) {
                const uint64_t dq = tc::sdesc_k(sq + t * C::OP), dk = tc::sdesc_sw128(sa(slots + uniform(step % C::SLOTS) * C::OP), 16, D * 16);
                if (elect()) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint64_t oq = (uint64_t)((k / 4 * C::HALF + k % 4 * 32) >> 4), ok = (uint64_t)((k / 4 * 1024 + k % 4 * 32) >> 4);
                        tc::mma_ss(tb + t * 128, dq + oq, dk + ok, IDS, k != 0);
                    }
                    tc::commit(&sfull[t]);
                }
                __syncwarp();
            };
            auto values = [&](int t, int step, bool first) {
                const uint64_t dv = tc::sdesc_sw128(sa(slots + uniform(step % C::SLOTS) * C::OP), 1024, D * 16);
                // P comes in two halves of 64 positions, each with its barrier (the second may come before the first is seen)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!wait(&pready[2 * t + h], cnt[t] & 1)) return false;
                    tc::fence_after();
                    if (elect()) {
#pragma unroll
                        for (int k = h * 4; k < h * 4 + 4; ++k)
                            tc::mma_ts(tb + 256 + t * 128, tb + t * 128 + k * 8, dv + (uint64_t)(k * D * 32 >> 4), IDO, !(first && k == 0));
                        if (h == 1) tc::commit(&pvdone[t]);
                    }
                    __syncwarp();
                }
                ++cnt[t];
                return true;
            };
            // a slot is free once the products that read it are done
            auto release = [&](int step, bool used) {
                if (elect()) {
                    if (used) tc::commit(&empty[step % C::SLOTS]);
                    else mbar_arrive(&empty[step % C::SLOTS]);
                }
                __syncwarp();
            };
            do {
                const int n0 = n_of(0), n1 = n_of(1);
                if (!(ok = wait(qfull, item & 1) && wait_slot(it))) break;
                tc::fence_after();
                if (n0 > 0) scores(0, it);
                if (n1 > 0) scores(1, it);
                release(it, n0 > 0 || n1 > 0);
                // The item's last scores have been issued: the next item's rows of q may come once they are done, while
                // this item's last values are still to do.
                auto release_q = [&]() {
                    if (elect()) {
                        if (n0 > 0 || n1 > 0) tc::commit(qempty);
                        else mbar_arrive(qempty);
                    }
                    __syncwarp();
                };
                if (w.n == 1) release_q();
                for (int u = 0; ok && u < w.n; ++u, it += 2) {
                    const bool more = u + 1 < w.n;
                    if (!(ok = wait_slot(it + 1))) break;
                    tc::fence_after();
                    if (u < n0 && !(ok = values(0, it + 1, u == 0))) break;
                    if (more && !(ok = wait_slot(it + 2))) break;
                    tc::fence_after();
                    if (u + 1 < n0) scores(0, it + 2);
                    if (u < n1 && !(ok = values(1, it + 1, u == 0))) break;
                    release(it + 1, u < n0 || u < n1);
                    if (u + 1 < n1) scores(1, it + 2);
                    if (more) release(it + 2, u + 1 < n0 || u + 1 < n1);
                    if (u + 2 == w.n) release_q();
                }
                ++item;
            } while (ok && w.next(a));
            // Whoever's wait ran out: the products issued so far are done before their tensor memory and shared memory are
            // given back.
            if (elect()) tc::commit(last);
            __syncwarp();
            wait_done(last, 0);
        }
    } else {  // rows of tile t: warp's lanes are tensor-memory lanes 32 (warp % 4) ..
        const int t = warp >= 6, q4 = warp & 3, i = q4 * 32 + lane;
        const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
        const uint32_t S = tb + t * 128 + lanes, O = tb + 256 + t * 128 + lanes;
        int cnt = 0;
        int v_it = 1;  // ring step of the unit's V
        bool ok = true;
        do {
            const int tok = (w.p.tile * 2 + t) * tq + i / group;
            const bool valid = i < tq * group && tok < w.q;
            const int lim = valid ? row_limit(a.s, w.q, w.kv, tok) : 0;
            const int n = n_of(t);
            float m = -INFINITY, l = 0.0f;
            for (int u = 0; ok && u < n; ++u, ++cnt) {
                ok = bounded_wait<QUICK>(&sfull[t], cnt & 1, abort_flag, a);
                ok = __all_sync(~0u, ok);
                if (!ok) break;
                tc::fence_after();
                const int p0 = (w.p.unit + u) * kLongUnit;
                const int left = lim - p0;  // positions of this unit that the row attends
                const bool cut = __any_sync(~0u, left < kLongUnit);
                // 64 scores in registers at a time: the second half is read for the maximum, and again after the first is done
                float x[64];
                auto half = [&](int h) {
                    ld64w(S + h * 64, x);
                    if (cut) {
#pragma unroll
                        for (int j = 0; j < 64; ++j) x[j] = h * 64 + j < left ? x[j] : -INFINITY;
                    }
                };
                auto top_of = [&]() {
                    float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                    for (int j = 4; j < 60; j += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k) mx[k] = fmaxf(fmaxf(mx[k], x[j + 2 * k]), x[j + 2 * k + 1]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], x[60 + k]);
                    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                };
                half(1);
                float top = top_of();
                half(0);
                top = fmaxf(top, top_of());
                // (the exponents take the product with the scale whole: in f16 none may come out above the rounded maximum)
                top = top == -INFINITY ? top : Cvt<T>::UP_LONG > 0.0f ? __fmul_ru(top, a.scale) : top * a.scale;
                const bool grow = u == 0 || top - m > Cvt<T>::UP_LONG + Cvt<T>::LAG;
                if (u == 0) {
                    m = base_of(top, Cvt<T>::UP_LONG);
                } else if (__any_sync(~0u, grow)) {
                    // (in f16, which has little room, every row of the warp whose maximum has grown joins in)
                    const bool up = Cvt<T>::UP_LONG > 0.0f ? top - m > Cvt<T>::UP_LONG : grow;
                    const float next = base_of(top, Cvt<T>::UP_LONG), f = up ? exp2_approx(m - next) : 1.0f;
                    if (up) m = next;
                    l *= f;
                    ok = __all_sync(~0u, bounded_wait<QUICK>(&pvdone[t], (cnt - 1) & 1, abort_flag, a));
                    if (!ok) break;
                    tc::fence_after();
#pragma unroll 1
                    for (int d = 0; d < D; d += 16) {
                        uint32_t r[16];
                        ld16w(O + d, r);
#pragma unroll
                        for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
                        tc::st16(O + d, r);
                    }
                }
                if (p0 + kLongUnit > w.kv) {  // V rows behind the last position: whatever the page holds must not reach the sums
                    const int it = v_it + 2 * u, s = it % C::SLOTS;
                    ok = __all_sync(~0u, bounded_wait<QUICK>(&full[s], (it / C::SLOTS) & 1, abort_flag, a));
                    if (!ok) break;
                    const int r0 = max(w.kv - p0, 0);
                    for (int e = i; e < (kLongUnit - r0) * (D / 8); e += 128) {
                        const int r = r0 + e / (D / 8), ch = e % (D / 8);
                        *reinterpret_cast<uint4 *>(slots + s * C::OP + kv_offset<D>(r, ch)) = make_uint4(0, 0, 0, 0);
                    }
                    tc::fence_proxy_async();
                    __syncwarp();
                }
                const float base = m == -INFINITY ? 0.0f : m;
                const unsigned long long scale2 = two(a.scale, a.scale), base2 = two(-base, -base);
                unsigned long long sum[2] = {0ull, 0ull};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h == 1) half(1);
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        uint32_t pk[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int e = g * 32 + 2 * j;
                            float pa, pb;
                            halves(fma2(two(x[e], x[e + 1]), scale2, base2), pa, pb);
                            pa = exp2_approx(pa);
                            pb = exp2_approx(pb);
                            sum[j & 1] = add2(sum[j & 1], two(pa, pb));
                            pk[j] = Cvt<T>::pack(pa, pb);
                        }
                        tc::st16(S + h * 32 + g * 16, pk);
                    }
                    tc::st_wait();
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&pready[2 * t + h]);
                }
                float s0, s1;
                halves(add2(sum[0], sum[1]), s0, s1);
                l += s0 + s1;
            }
            // the item's rows
            if (ok && n > 0) ok = __all_sync(~0u, bounded_wait<QUICK>(&pvdone[t], (cnt - 1) & 1, abort_flag, a));
            if (!ok) break;
            tc::fence_after();
            const bool whole = w.whole();
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            const int slot = 2 * c + w.slot(), row = t * 128 + i;
            float *part = a.part + slot * a.slot_floats;
            T *dst = static_cast<T *>(a.out) + (int64_t)(w.q0 + tok) * a.o_row + (w.p.head * group + i % group) * a.o_head;
#pragma unroll 2
            for (int d = 0; d < D; d += 16) {
                uint32_t r[16] = {};
                float o[16];
                if (n > 0) ld16w(O + d, r);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __uint_as_float(r[e]);
                if (valid && whole) {
#pragma unroll
                    for (int e = 0; e < 16; e += 8)
                        *reinterpret_cast<uint4 *>(dst + d + e) =
                            make_uint4(Cvt<T>::pack(o[e] * inv, o[e + 1] * inv), Cvt<T>::pack(o[e + 2] * inv, o[e + 3] * inv),
                                       Cvt<T>::pack(o[e + 4] * inv, o[e + 5] * inv), Cvt<T>::pack(o[e + 6] * inv, o[e + 7] * inv));
                } else if (valid) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<float4 *>(part + (int64_t)row * D + d + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
                __syncwarp();
            }
            tc::fence_before();
            if (!whole) {
                if (valid) reinterpret_cast<float2 *>(part + (int64_t)a.rows * D)[row] = make_float2(m, l);
                if (i == 0 && t == 0) a.meta[slot] = make_int4(w.ends() ? 3 : 1, w.r, w.p.head, w.p.tile);
            }
            v_it += 2 * w.n;
        } while (w.next(a));
        tc::st_wait();
    }
    tc::fence_before();
    __syncthreads();
    if (warp == 0) {
        tc::fence_after();
        tc::dealloc(tb, 512);
    }
}

// q as [rows][K/V heads][group][head_dim]: a box is TQ tokens' rows of one K/V
// head, 64 elements wide, in the order of the tile's rows.
bool q_map(CUtensorMap *m, const AttendArgs &a, int d) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const int tq = a.s.tile / 2;
    const int64_t head = a.s.group * a.s.n_kv > 1 ? a.q_head : d, row = a.total_q > 1 ? a.q_row : d;
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)a.s.group, (cuuint64_t)a.s.n_kv, (cuuint64_t)a.total_q};
    const cuuint64_t strides[3] = {(cuuint64_t)head * 2, (cuuint64_t)(head * a.s.group) * 2, (cuuint64_t)row * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)a.s.group, 1, (cuuint32_t)tq}, es[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void *>(a.q), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool QUICK>
cudaError_t launch(const PoolMap &kv, const AttendArgs &a, int parts, cudaStream_t s) {
    LongMaps maps;
    std::memset(&maps, 0, sizeof(maps));
    maps.kv = kv;
    if (!q_map(&maps.q, a, D)) return cudaErrorInvalidValue;
    using C = LongCfg<D>;
    static std::atomic<bool> set[64];  // attributes, per device
    const int device = dev::current() & 63;
    if (!set[device].load(std::memory_order_acquire)) {
        cudaError_t e = dev::smem(attend_long_kernel<T, D, QUICK>, C::SMEM);
        if (e == cudaSuccess) e = dev::whole_smem(attend_long_kernel<T, D, QUICK>);
        if (e != cudaSuccess) return e;
        set[device].store(true, std::memory_order_release);
    }
    return launch_pdl(attend_long_kernel<T, D, QUICK>, dim3(parts), dim3(LONG_THREADS), C::SMEM, s, maps, a);
}

template <typename T, int D>
cudaError_t launch(const PoolMap &kv, const AttendArgs &a, int parts, cudaStream_t s) {
    return a.quick ? launch<T, D, true>(kv, a, parts, s) : launch<T, D, false>(kv, a, parts, s);
}

}  // namespace

cudaError_t attend_long(const PoolMap &kv, const AttendArgs &a, bool bf16, int head_dim, int parts, cudaStream_t s) {
    if (head_dim == 64) return bf16 ? launch<__nv_bfloat16, 64>(kv, a, parts, s) : launch<__half, 64>(kv, a, parts, s);
    return bf16 ? launch<__nv_bfloat16, 128>(kv, a, parts, s) : launch<__half, 128>(kv, a, parts, s);
}

}  // namespace serve
}  // namespace kg
