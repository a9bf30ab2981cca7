// kg_pool_sched.h — how kg_pool_attend_dev's work is cut: plain integer
// arithmetic, used by the kernels and, compiled as C++, by a CPU test.
//
// A request whose rows (new tokens x query heads per K/V head) fit kShortRows
// is "short": one item per K/V head, units of `unit` positions. The others
// are "long": one item per (K/V head, tile of tokens), units of kLongUnit
// positions up to the tile's last attended one. An item always has a unit, so
// that rows which attend nothing get their zeros. The units of all items in
// order (request, head, tile, unit) form one line that is cut into equal parts,
// one per CTA: a part is a run of units that may begin and end inside an item.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define KG_HD __host__ __device__ __forceinline__
#else
#define KG_HD inline
#endif

namespace kg {
namespace serve {

constexpr int kShortRows = 64, kLongUnit = 128;
constexpr int kMaxKv = 2147483647 - 256;  // a unit that begins before the last position ends inside 31 bits

struct Shape {
    int group;      // query heads per K/V head
    int n_kv;       // K/V heads
    int tile;       // tokens of a long item
    int causal;
    int unit;       // positions of a short item's unit
};

KG_HD bool lengths_ok(int q0, int q1, int kv, int total_q, int64_t room) {
    return q0 >= 0 && q1 >= q0 && q1 <= total_q && kv >= 0 && kv <= room;
}
KG_HD bool is_short(const Shape &s, int q) { return (int64_t)q * s.group <= kShortRows; }

// units of one head's item of a short request (0: none)
KG_HD int short_units(const Shape &s, int q, int kv) {
    if (q == 0 || !is_short(s, q)) return 0;
    return kv > 0 ? (kv - 1) / s.unit + 1 : 1;
}
KG_HD int long_tiles(const Shape &s, int q) { return q == 0 || is_short(s, q) ? 0 : (q - 1) / s.tile + 1; }
// positions that token t's row attends: [0, limit)
KG_HD int row_limit(const Shape &s, int q, int kv, int t) {
    if (!s.causal) return kv;
    const int64_t n = (int64_t)kv - q + t + 1;
    return n < 0 ? 0 : (int)n;
}
KG_HD int long_units(const Shape &s, int q, int kv, int i) {
    const int64_t end = (int64_t)(i + 1) * s.tile;
    const int n = row_limit(s, q, kv, (int)(end < q ? end : q) - 1);
    return n > 0 ? (n - 1) / kLongUnit + 1 : 1;
}
// sum over i < n of floor((a i + b) / 128), a > 0, b >= 0: the terms repeat, but for a step, after 128 / gcd(a, 128)
KG_HD int64_t sum_of_units(int n, int a, int64_t b) {
    const int low = a & -a, period = low >= 128 ? 1 : 128 / low;
    const int64_t rise = (int64_t)a * period / 128, rounds = n / period;
    const int rest = n % period;
    int64_t once = 0, tail = 0;
    for (int i = 0; i < period && i < n; ++i) {
        const int64_t f = ((int64_t)a * i + b) >> 7;
        once += f;
        if (i < rest) tail += f;
    }
    if (rounds == 0) return tail;
    return rounds * once + period * rise * (rounds * (rounds - 1) / 2) + tail + rest * rounds * rise;
}
// units of the first n tiles of one head's long items
KG_HD int64_t long_units_before(const Shape &s, int q, int kv, int n) {
    const int tiles = long_tiles(s, q);
    int64_t sum = 0;
    if (n >= tiles && tiles > 0) {  // the last tile may be short
        sum = long_units(s, q, kv, tiles - 1);
        n = tiles - 1;
    }
    if (n <= 0) return sum;
    if (!s.causal) return sum + (int64_t)n * long_units(s, q, kv, 0);
    // tile i attends base + (i + 1) tile positions; where that is not positive it has one unit all the same
    const int64_t base = (int64_t)kv - q;
    int none = base < 0 ? (int)(-base / s.tile) : 0;
    none = none < n ? none : n;
    return sum + none + sum_of_units(n - none, s.tile, base + (int64_t)(none + 1) * s.tile + 127);
}
KG_HD int64_t long_units_of_head(const Shape &s, int q, int kv) { return long_units_before(s, q, kv, long_tiles(s, q)); }
// units of a whole request in the line of short or of long items
KG_HD int64_t request_units(const Shape &s, bool is_long, int q, int kv) {
    return (is_long ? long_units_of_head(s, q, kv) : short_units(s, q, kv)) * s.n_kv;
}
// items of a request
KG_HD int64_t request_items(const Shape &s, bool is_long, int q, int kv) {
    return (is_long ? long_tiles(s, q) : q > 0 && is_short(s, q) ? 1 : 0) * (int64_t)s.n_kv;
}
// Parts of a line: at most `most`, of at least `least` units each, but one for every item where there are so few (a CTA
// takes its items one after the other).
KG_HD int parts_of(int64_t units, int64_t items, int most, int least) {
    const int64_t n = (units + least - 1) / least, m = n > items ? n : items;
    return (int)(m < most ? m : most);
}
// the first unit of part c of `parts` (in 32 bits where they suffice: 64-bit divisions are slow on the device)
KG_HD int64_t part_begin(int64_t units, int c, int parts) {
    if (units <= 4194303) {  // units % parts * c stays below 512 * 512
        const uint32_t n = (uint32_t)units, p = (uint32_t)parts, k = (uint32_t)c;
        return n / p * k + n % p * k / p;
    }
    return units / parts * c + units % parts * c / parts;
}

// A place in the line: item (head, tile) of a request, its first unit here and its length.
struct Place {
    int head, tile, unit, units;
};
KG_HD Place place_of(const Shape &s, bool is_long, int q, int kv, int64_t off) {
    Place p;
    if (!is_long) {
        p.units = short_units(s, q, kv);
        if (off <= 0x7fffffff) {
            p.head = (int)((uint32_t)off / (uint32_t)p.units);
            p.unit = (int)((uint32_t)off % (uint32_t)p.units);
        } else {
            p.head = (int)(off / p.units);
            p.unit = (int)(off % p.units);
        }
        p.tile = 0;
        return p;
    }
    const int64_t per = long_units_of_head(s, q, kv);
    p.head = (int)(off / per);
    const int64_t rest = off % per;
    int lo = 0, hi = long_tiles(s, q) - 1;  // the last tile whose units before it are at most `rest`
    while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (long_units_before(s, q, kv, mid) <= rest) lo = mid;
        else hi = mid - 1;
    }
    p.tile = lo;
    p.units = long_units(s, q, kv, lo);
    p.unit = (int)(rest - long_units_before(s, q, kv, lo));
    return p;
}

}  // namespace serve
}  // namespace kg
