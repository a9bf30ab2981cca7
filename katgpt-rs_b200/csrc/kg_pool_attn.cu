// kg_pool_attn.cu — kg_pool_attend_dev: attention of new rows over a paged K/V
// pool, ragged over requests.
//
// One pass over the positions with a running maximum m (less a constant in f16: Cvt) and
// sum l per row:
//   o = sum_j 2^(s_j - m) v_j,  l = sum_j 2^(s_j - m),  s_j = scale log2(e) q.k_j
// A part of the positions gives (o, m, l); parts of one item join as
//   M = max m,  out = sum 2^(m - M) o / sum 2^(m - M) l.
// The work is one line of units cut into equal parts (kg_pool_sched.h), so that
// one long sequence fills the device as well as many short ones, and the lengths
// are read on the device.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <cstring>
#include <type_traits>

#include "kg_dev.cuh"
#include "kg_pdl.cuh"
#include "kg_pool_attn.cuh"
#include "kg_serve.h"

namespace kg {
namespace serve {
namespace {

using namespace as;

// ---------------------------------------------------------------------------
// Short requests (at most 64 rows: single tokens, draft paths) on mma.sync:
// rows (token, query head of the group) x positions. Bound by the bytes of K and
// V; a producer warp keeps a ring of three 32 KB stages (64 positions of 128
// dimensions, 128 of 64) filled by TMA, one box per page, and four warps split a
// stage by rows (groups of 16) and by positions, 32 at a time where they have them.
// Each keeps its own running maximum and sum, joined at the end of the item. 64 single
// tokens over 4.2 K positions of 32 heads of 128 (4.36 GB): 641 us, 104% of the copy
// rate; 32 over 0.3 to 16 K positions of 8 heads: 173 us (89%); 64 over 1.1 K positions of
// 12 heads of 64: 50 us (67%), with pages of 16 or 128 rows alike, 5 us of it before the
// first bytes are there and 6 us the joining kernel.
constexpr int SHORT_THREADS = 160, SHORT_LEAST = 2;  // (of 1, 2 and 4 units a part, 8 x 500 positions: 19, 13 and 13 us)

template <int D>
struct ShortCfg {
    static constexpr int UNIT = 64 * 128 / D;       // positions
    static constexpr int OP_BYTES = UNIT * D * 2;  // K or V of a stage
    static constexpr int STAGES = 3;
    static constexpr int SCRATCH = 4 * 16 * 36 * 4;
    static constexpr int SMEM = 1024 + STAGES * 2 * OP_BYTES + SCRATCH + 4 * 16 * 2 * 4 + 2 * STAGES * 8 + 16;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void bar_consumers() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <typename T, int D, bool QUICK>
__global__ void __launch_bounds__(SHORT_THREADS) attend_short_kernel(const __grid_constant__ PoolMap maps, const AttendArgs a,
                                                                   int after_long) {
    using C = ShortCfg<D>;
    extern __shared__ __align__(1024) uint8_t raw[];
    uint8_t *sm = raw + ((1024u - (sa(raw) & 1023u)) & 1023u);
    float *scratch = reinterpret_cast<float *>(sm + C::STAGES * 2 * C::OP_BYTES);  // [4 warps][16 rows][36]
    float2 *stat = reinterpret_cast<float2 *>(scratch + 4 * 16 * 36);              // [4 warps][16 rows] (max, sum)
    uint64_t *full = reinterpret_cast<uint64_t *>(stat + 4 * 16), *empty = full + C::STAGES;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(empty + C::STAGES);
    __shared__ long long part_sm[2 * (SHORT_THREADS / 32) + 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 4);
        }
        *abort_flag = 0;
        mbar_fence_init();
        prefetch_map(&maps.k);
        prefetch_map(&maps.v);
    }
    // Behind the long requests' kernel this one starts as soon as that one's CTAs all run (they have waited for what came
    // before), and waits for it at its own end: the two share the device, and what follows waits for both.
    if (!after_long) pdl_wait();
    int req;
    long long off, units;
    find_part<SHORT_THREADS, false>(a, c, gridDim.x, SHORT_LEAST, part_sm, req, off, units);  // (synchronises)
    if (threadIdx.x < 2) a.meta[2 * c + threadIdx.x].x = 0;
    __syncthreads();
    if (units == 0) {
        if (after_long) pdl_wait();
        return;
    }
    Walk<false> w;
    w.start(a, req, off, units);

    Ring<QUICK> ring{full, empty, 2 * C::OP_BYTES, abort_flag, a};
    if (warp == 4) {  // producer: lane i loads box i of a unit
        const int rows = min(a.page_size, kBoxRows), pages = C::UNIT / rows, boxes = pages * 2;
        const int piece = lane % pages, which = lane / pages;
        const CUtensorMap *tm = which ? &maps.v : &maps.k;
        const int dst = which * C::OP_BYTES + piece * rows * D * 2;
        int it = 0;
        bool ok = true;
        do {
            for (int u = 0; u < w.n; ++u, ++it) {
                const int s = it % C::STAGES, pos = (w.p.unit + u) * C::UNIT + piece * rows;
                int place = maps.outside;
                if (lane < boxes && pos < w.kv) {
                    const int e = a.table[(int64_t)w.r * a.width + pos / a.page_size];
                    if (e >= 0 && e < a.n_pages) place = e * maps.page_step + w.p.head * maps.head_step;
                    else reject(a.err);
                }
                if (lane == 0) ok = ring_claim(ring, C::STAGES, it);
                ok = __shfl_sync(~0u, ok, 0);
                if (!ok) break;
                if (lane < boxes)
                    tma_load_5d(sm + s * 2 * C::OP_BYTES + dst, tm, pos % a.page_size / 8, place, &full[s]);
            }
        } while (ok && w.next(a));
        ring_drain(ring, C::STAGES, it);
        if (after_long) pdl_wait();
        return;
    }

    const int gid = lane >> 2, tig = lane & 3;
    bool ok = true;
    int it = 0;
    do {
        const int rows = w.q * a.s.group, wm = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;  // row groups
        const int rg = warp % wm, pg = warp / wm;
        // Q fragments of rows 16 rg + gid and + 8
        uint32_t qf[D / 16][4];
        int lim[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = rg * 16 + gid + 8 * i, t = row / a.s.group, h = w.p.head * a.s.group + row % a.s.group;
            const bool in = row < rows;
            lim[i] = in ? row_limit(a.s, w.q, w.kv, t) : 0;
            const uint32_t *src = reinterpret_cast<const uint32_t *>(static_cast<const T *>(a.q) + (w.q0 + t) * a.q_row + h * a.q_head);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qf[k][i] = in ? __ldg(src + k * 8 + tig) : 0u;
                qf[k][i + 2] = in ? __ldg(src + k * 8 + tig + 4) : 0u;
            }
        }
        float o[D / 8][4];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        for (int u = 0; u < w.n; ++u, ++it) {
            const int s = it % C::STAGES;
            // (a wait that gave up skips the work, not the barriers below)
            ok = ring_take(ring, C::STAGES, it, ok);
            uint8_t *st = sm + s * 2 * C::OP_BYTES;
            bool wrote = false;
            const int chunk = C::UNIT / 4 * wm, p_end = (pg + 1) * chunk, unit0 = (w.p.unit + u) * C::UNIT;
            // positions p0 .. p0 + 16 NB of the stage
            auto step = [&](auto nb, int p0) {
                constexpr int NB = decltype(nb)::value;
                const int pos0 = unit0 + p0;
                if (pos0 + 16 * NB > w.kv) {  // rows behind the last position: whatever the page holds must not reach the sums
                    for (int i = lane; i < 16 * NB * (D / 8); i += 32) {
                        const int r = i / (D / 8), ch = i % (D / 8);
                        if (pos0 + r >= w.kv)
                            *reinterpret_cast<uint4 *>(st + C::OP_BYTES + kv_offset<D>(p0 + r, ch)) = make_uint4(0, 0, 0, 0);
                    }
                    wrote = true;
                    __syncwarp();
                }
                float sc[2 * NB][4] = {};
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const int r = p0 + b * 16 + (lane & 7) + ((lane >> 4) << 3), ch = k * 2 + ((lane >> 3) & 1);
                        uint32_t kf[4];
                        ldsm4(sa(st) + kv_offset<D>(r, 0) + (ch >> 3) * 1024 + (((ch & 7) ^ (r & 7)) << 4), kf);
                        mma16816<T>(sc[2 * b], qf[k], kf[0], kf[1]);
                        mma16816<T>(sc[2 * b + 1], qf[k], kf[2], kf[3]);
                    }
                uint32_t pf[NB][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float x[4 * NB], mx = -INFINITY;
#pragma unroll
                    for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            x[n * 2 + e] = pos0 + n * 8 + tig * 2 + e < lim[i] ? sc[n][i * 2 + e] * a.scale : -INFINITY;
                            mx = fmaxf(mx, x[n * 2 + e]);
                        }
                    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
                    const float mn = fmaxf(m[i], base_of(mx, Cvt<T>::UP));
                    if (__any_sync(~0u, mn != m[i])) {
                        const float f = mn == -INFINITY ? 1.0f : exp2_approx(m[i] - mn);
                        l[i] *= f;
#pragma unroll
                        for (int n = 0; n < D / 8; ++n) {
                            o[n][i * 2] *= f;
                            o[n][i * 2 + 1] *= f;
                        }
                        m[i] = mn;
                    }
                    const float base = mn == -INFINITY ? 0.0f : mn;
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4 * NB; ++e) {
                        x[e] = exp2_approx(x[e] - base);
                        sum += x[e];
                    }
                    l[i] += sum;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        pf[b][i] = Cvt<T>::pack(x[4 * b], x[4 * b + 1]);
                        pf[b][i + 2] = Cvt<T>::pack(x[4 * b + 2], x[4 * b + 3]);
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const int r = p0 + b * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), ch = k * 2 + (lane >> 4);
                        uint32_t vf[4];
                        ldsm4t(sa(st) + C::OP_BYTES + kv_offset<D>(r, 0) + (ch >> 3) * 1024 + (((ch & 7) ^ (r & 7)) << 4), vf);
                        mma16816<T>(o[2 * k], pf[b], vf[0], vf[1]);
                        mma16816<T>(o[2 * k + 1], pf[b], vf[2], vf[3]);
                    }
            };
            if (ok) {
                if (D == 128 && chunk == 16) {
                    if (unit0 + pg * 16 < w.kv) step(std::integral_constant<int, 1>(), pg * 16);
                } else {
                    for (int p0 = pg * chunk; p0 < p_end && unit0 + p0 < w.kv; p0 += 32) step(std::integral_constant<int, 2>(), p0);
                }
            }
            if (wrote) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before TMA writes the stage again
            __syncwarp();
            if (lane == 0) ring_free(ring, C::STAGES, it, ok);
        }
        // join the warps that share rows and write the item
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(~0u, l[i], 1);
            l[i] += __shfl_xor_sync(~0u, l[i], 2);
            if (tig == 0) stat[warp * 16 + gid + 8 * i] = make_float2(m[i], l[i]);
        }
        bar_consumers();
        auto top_of = [&](int g, int r) {
            float x = -INFINITY;
            for (int k = g; k < 4; k += wm) x = fmaxf(x, stat[k * 16 + r].x);
            return x;
        };
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) f[i] = m[i] == -INFINITY ? 0.0f : exp2_approx(m[i] - top_of(rg, gid + 8 * i));
        const bool whole = w.whole();
        const int slot = 2 * c + w.slot();
        float *part = a.part + slot * a.slot_floats;
        // `width` dims of every row at a time, as the scratch holds: all of them where a request has few rows
        const int few = rows <= 4, width = few ? D : 32, pitch = few ? D : 36, cap = few ? 4 : 16;
        for (int d0 = 0; d0 < D; d0 += width) {
            float *mine = scratch + warp * cap * pitch;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
                if (few || n / 4 == d0 / 32)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (gid + 8 * i < cap)
                            *reinterpret_cast<float2 *>(mine + (gid + 8 * i) * pitch + (few ? n : n & 3) * 8 + tig * 2) =
                                make_float2(o[n][i * 2] * f[i], o[n][i * 2 + 1] * f[i]);
            bar_consumers();
            for (int i = threadIdx.x; i < rows * (width / 4); i += 128) {
                const int row = few ? i / (D / 4) : i >> 3, d = (few ? i % (D / 4) : i & 7) * 4, g = row >> 4, r = row & 15;
                float4 sum = make_float4(0, 0, 0, 0);
                for (int k = g; k < 4; k += wm) {
                    const float4 x = *reinterpret_cast<const float4 *>(scratch + (k * cap + r) * pitch + d);
                    sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
                }
                const float top = top_of(g, r);
                float total = 0.0f;
                for (int k = g; k < 4; k += wm) {
                    const float2 x = stat[k * 16 + r];
                    total += x.x == -INFINITY ? x.y : x.y * exp2_approx(x.x - top);  // (there a sum is 0, or NaN as its scores)
                }
                if (whole) {
                    const float inv = total > 0.0f ? 1.0f / total : 0.0f;
                    T *dst = static_cast<T *>(a.out) + (w.q0 + row / a.s.group) * a.o_row +
                             (w.p.head * a.s.group + row % a.s.group) * a.o_head + d0 + d;
                    *reinterpret_cast<uint2 *>(dst) =
                        make_uint2(Cvt<T>::pack(sum.x * inv, sum.y * inv), Cvt<T>::pack(sum.z * inv, sum.w * inv));
                } else {
                    *reinterpret_cast<float4 *>(part + (int64_t)row * D + d0 + d) = sum;
                    if (d0 == 0 && d == 0) reinterpret_cast<float2 *>(part + (int64_t)a.rows * D)[row] = make_float2(top, total);
                }
            }
            bar_consumers();
        }
        if (!whole && threadIdx.x == 0) a.meta[slot] = make_int4(w.ends() ? 3 : 1, w.r, w.p.head, 0);
    } while (w.next(a));
    if (after_long) pdl_wait();
}

// Joins the parts of the items that were cut, of both kernels: two blocks (eight for
// the long requests' parts) look after the item that begins in a part and ends beyond
// it, eight rows at a time. (A block for every eight rows there could be, 14 thousand
// mostly empty ones, took 15 us.)
// Few parts: a warp a row; many (a lone long sequence): the block's warps share a
// row's parts. Part sums are added in a fixed order, so results do not depend on
// timing.
constexpr int JOIN_ROWS = 8, JOIN_FEW = 16, JOIN_SHORT = 2, JOIN_LONG = 8;

template <typename T, int D>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendArgs sh, int short_parts, const AttendArgs lo) {
    pdl_wait();
    __shared__ int s_last;
    __shared__ float4 sums[8][32];
    __shared__ float part_l[8];
    const bool is_long = (int)blockIdx.x >= short_parts * JOIN_SHORT;
    const AttendArgs &a = is_long ? lo : sh;
    const int per = is_long ? JOIN_LONG : JOIN_SHORT, x = is_long ? blockIdx.x - short_parts * JOIN_SHORT : blockIdx.x;
    const int c = x / per, parts = is_long ? (gridDim.x - short_parts * JOIN_SHORT) / JOIN_LONG : short_parts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int4 me = a.meta[2 * c + 1];
    if (me.x == 0) return;
    int q0, q, kv;
    req_len(a, me.y, q0, q, kv);
    const int group = a.s.group, tq = a.s.tile / 2, rows = is_long ? 256 : q * group;
    if (x % per * JOIN_ROWS >= rows) return;
    if (threadIdx.x == 0) {
        int e = c + 1;
        while (e < parts - 1 && a.meta[2 * e].x == 1) ++e;
        s_last = e;
    }
    __syncthreads();
    const int n = s_last - c + 1;
    auto slot = [&](int i) { return a.part + (i == 0 ? 2 * c + 1 : 2 * (c + i)) * a.slot_floats; };
    constexpr int PER = D / 32;  // dims of a lane
    auto each = [&](int row) {   // its token, or -1
        const int i = is_long ? row & 127 : row;
        const int tok = is_long ? (me.w * 2 + (row >> 7)) * tq + i / group : i / group;
        return row >= rows || (is_long && i >= tq * group) || tok >= q ? -1 : tok;
    };
    auto sum_of = [&](int row, int first, int step, float (&o)[PER], float &l) {
        auto stat_of = [&](int k) { return reinterpret_cast<const float2 *>(slot(k) + (int64_t)a.rows * D)[row]; };
        float top = -INFINITY;
        for (int k = lane; k < n; k += 32) top = fmaxf(top, stat_of(k).x);
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
#pragma unroll 4
        for (int k = first; k < n; k += step) {
            const float2 s = stat_of(k);
            if (s.x == -INFINITY && s.y == 0.0f) continue;  // nothing was attended there (a sum that is NaN is to be seen)
            const float f = exp2_approx(s.x - top);
            const float *p = slot(k) + (int64_t)row * D + lane * PER;
            l += s.y * f;
#pragma unroll
            for (int e = 0; e < PER; ++e) o[e] += p[e] * f;
        }
    };
    auto write = [&](int row, int tok, const float (&o)[PER], float l) {
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        const int i = is_long ? row & 127 : row;
        T *dst = static_cast<T *>(a.out) + (int64_t)(q0 + tok) * a.o_row + (me.z * group + i % group) * a.o_head + lane * PER;
#pragma unroll
        for (int e = 0; e < PER; e += 2) reinterpret_cast<uint32_t *>(dst)[e / 2] = Cvt<T>::pack(o[e] * inv, o[e + 1] * inv);
    };
    for (int row0 = x % per * JOIN_ROWS; row0 < rows; row0 += per * JOIN_ROWS) {
        if (n <= JOIN_FEW) {
            const int row = row0 + warp, tok = each(row);
            if (tok < 0) continue;
            float o[PER] = {}, l = 0.0f;
            sum_of(row, 0, 1, o, l);
            write(row, tok, o, l);
            continue;
        }
        for (int row = row0; row < row0 + JOIN_ROWS; ++row) {
            const int tok = each(row);
            if (tok < 0) continue;
            float o[PER] = {}, l = 0.0f;
            sum_of(row, warp, 8, o, l);
            sums[warp][lane] = make_float4(o[0], o[1], PER > 2 ? o[PER - 2] : 0.0f, PER > 2 ? o[PER - 1] : 0.0f);
            if (lane == 0) part_l[warp] = l;
            __syncthreads();
            if (warp == 0) {
                float t[PER] = {}, total = 0.0f;
                for (int k = 0; k < 8; ++k) {
                    const float4 v = sums[k][lane];
                    t[0] += v.x;
                    t[1] += v.y;
                    if (PER > 2) {
                        t[PER - 2] += v.z;
                        t[PER - 1] += v.w;
                    }
                    total += part_l[k];
                }
                write(row, tok, t, total);
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------------------
// Host

// The pool's maps (PoolMap); false when the driver refuses them.
bool pool_map(PoolMap &m, const kg_pool &p) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const int64_t unit = pool_unit(p), rs = p.row_stride;
    m.page_step = (int)(p.n_pages > 1 ? p.page_stride / unit : 0);
    m.head_step = (int)(p.n_kv_head > 1 ? p.head_stride / unit : 0);
    m.outside = (p.n_pages - 1) * m.page_step + (p.n_kv_head - 1) * m.head_step + 1;
    const cuuint64_t dims[5] = {64, 8, (cuuint64_t)p.head_dim / 64, (cuuint64_t)p.page_size / 8, (cuuint64_t)m.outside};
    const cuuint64_t strides[4] = {(cuuint64_t)rs * 2, 128, (cuuint64_t)rs * 16, (cuuint64_t)unit * 2};
    const cuuint32_t box[5] = {64, 8, (cuuint32_t)p.head_dim / 64, (cuuint32_t)std::min(p.page_size, kBoxRows) / 8, 1};
    const cuuint32_t es[5] = {1, 1, 1, 1, 1};
    for (int i = 0; i < 2; ++i)
        if (fn(i ? &m.v : &m.k, CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, i ? p.v : p.k, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, p.head_dim == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    return true;
}

// Workspace: [meta][part sums], for the short requests' kernel and then, where
// the rows of a call could make a request long, for the long requests'.
struct Space {
    int rows;
    bool may_long;
    int64_t slot_floats, long_at, long_floats, bytes;
};
Space space_of(const kg_pool &p, int n_head, int total_q) {
    Space s;
    const int64_t rows = (int64_t)total_q * (n_head / p.n_kv_head);
    s.rows = (int)std::min<int64_t>((rows + 15) / 16 * 16, kShortRows);
    s.slot_floats = (int64_t)s.rows * (p.head_dim + 2);
    s.may_long = rows > kShortRows;
    s.long_at = 2 * kMaxParts * ((int64_t)sizeof(int4) + s.slot_floats * 4);
    s.long_floats = 256 * (int64_t)(p.head_dim + 2);
    s.bytes = s.long_at + (s.may_long ? 2 * kMaxLongParts * ((int64_t)sizeof(int4) + s.long_floats * 4) : 0);
    return s;
}

template <typename T, int D, bool QUICK>
cudaError_t launch(const kg_pool &p, const Space &sp, AttendArgs a, void *workspace, cudaStream_t s) {
    PoolMap maps;
    std::memset(&maps, 0, sizeof(maps));
    if (!pool_map(maps, p)) return cudaErrorInvalidValue;
    using C = ShortCfg<D>;
    // per device, once: attributes and the CTAs that the device holds
    static std::atomic<int> held[64];
    const int device = dev::current() & 63;
    int parts = held[device].load(std::memory_order_acquire);
    cudaError_t e = cudaSuccess;
    if (parts == 0) {
        e = dev::smem(attend_short_kernel<T, D, QUICK>, C::SMEM);
        if (e == cudaSuccess) e = dev::whole_smem(attend_short_kernel<T, D, QUICK>);
        if (e == cudaSuccess) e = dev::whole_smem(attend_join_kernel<T, D>);
        if (e != cudaSuccess) return e;
        parts = std::min(kMaxParts, dev::sm_count() * dev::occupancy(attend_short_kernel<T, D, QUICK>, SHORT_THREADS, C::SMEM));
        held[device].store(parts, std::memory_order_release);
    }
    AttendArgs b = a;
    int long_parts = 0;
    if (sp.may_long) {
        b.meta = reinterpret_cast<int4 *>(static_cast<uint8_t *>(workspace) + sp.long_at);
        b.part = reinterpret_cast<float *>(b.meta + 2 * kMaxLongParts);
        b.slot_floats = sp.long_floats;
        b.rows = 256;
        long_parts = std::min(kMaxLongParts, dev::sm_count());
        e = attend_long(maps, b, std::is_same<T, __nv_bfloat16>::value, D, long_parts, s);
        if (e != cudaSuccess) return e;
    }
    a.meta = static_cast<int4 *>(workspace);
    a.part = reinterpret_cast<float *>(a.meta + 2 * kMaxParts);
    a.slot_floats = sp.slot_floats;
    a.rows = sp.rows;
    e = launch_pdl(attend_short_kernel<T, D, QUICK>, dim3(parts), dim3(SHORT_THREADS), C::SMEM, s, maps, a, (int)sp.may_long);
    if (e != cudaSuccess) return e;
    return launch_pdl(attend_join_kernel<T, D>, dim3(parts * JOIN_SHORT + long_parts * JOIN_LONG), dim3(256), 0, s, a, parts, b);
}
template <bool QUICK>
cudaError_t launch(const kg_pool &p, const Space &sp, const AttendArgs &a, void *ws, cudaStream_t s) {
    if (p.dtype == KG_DT_BF16) return p.head_dim == 64 ? launch<__nv_bfloat16, 64, QUICK>(p, sp, a, ws, s) : launch<__nv_bfloat16, 128, QUICK>(p, sp, a, ws, s);
    return p.head_dim == 64 ? launch<__half, 64, QUICK>(p, sp, a, ws, s) : launch<__half, 128, QUICK>(p, sp, a, ws, s);
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
    return kg::serve::space_of(*pool, n_head, total_q).bytes;
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
    const Space sp = space_of(*pool, n_head, total_q);
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
        if (workspace_bytes < sp.bytes) return fail(ctx, KG_ERR_INVALID_ARG, "attend: workspace smaller than kg_pool_attend_bytes");
        if (!(scale >= 0.0f && scale < INFINITY)) return fail(ctx, KG_ERR_INVALID_ARG, "attend: scale must be finite and not negative");
    }
    if (!ctx) return fail(ctx, KG_ERR_INVALID_ARG, "null context");
    if (!some) return KG_OK;
    DeviceGuard dg(ctx->device);
    if (dg.err != cudaSuccess) return cuda_fail(ctx, dg.err, "kg_pool_attend_dev");
    AttendArgs a;
    a.s = Shape{n_head / pool->n_kv_head, pool->n_kv_head, 2 * (128 / (n_head / pool->n_kv_head)), causal != 0, 64 * 128 / pool->head_dim};
    a.n_req = n_req;
    a.total_q = total_q;
    a.width = table_width;
    a.page_size = pool->page_size;
    a.n_pages = pool->n_pages;
    a.cu = cu_q;
    a.kv = kv_len;
    a.table = table;
    a.q = q;
    a.out = out;
    a.q_row = q_row_stride;
    a.q_head = q_head_stride;
    a.o_row = out_row_stride;
    a.o_head = out_head_stride;
    a.scale = std::max(scale * 1.4426950408889634f, FLT_MIN);  // (a masked score, -inf, times 0 would be NaN)
    a.err = ctx->serve_err;
    a.quick = ctx->serve_quick;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a.quick ? launch<true>(*pool, sp, a, workspace, s) : launch<false>(*pool, sp, a, workspace, s);
    return e == cudaSuccess ? KG_OK : cuda_fail(ctx, e, "kg_pool_attend_dev");
}

}  // extern "C"
