// Walks the cut of kg_pool_attend_dev's work (kg_pool_sched.h) on the CPU: every unit of every item belongs to exactly
// one part, in order, and a part is found from its number alone.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../katgpt-rs_b200/csrc/kg_pool_sched.h"

using namespace kg::serve;

static unsigned long long state = 88172645463325252ull;
static int rnd(int n) {
    state ^= state << 13;
    state ^= state >> 7;
    state ^= state << 17;
    return (int)(state % (unsigned)n);
}
#define CHECK(x)                                                   \
    do {                                                           \
        if (!(x)) {                                                \
            std::printf("line %d: %s\n", __LINE__, #x);            \
            return 1;                                              \
        }                                                          \
    } while (0)

int main() {
    const int groups[] = {1, 2, 3, 4, 5, 7, 8, 16, 33, 64};
    for (int trial = 0; trial < 3000; ++trial) {
        Shape s;
        s.group = groups[rnd(10)];
        s.n_kv = 1 + rnd(4);
        s.tile = 2 * (128 / s.group);
        s.causal = rnd(2);
        s.unit = rnd(2) ? 64 : 128;
        const int n_req = 1 + rnd(12);
        std::vector<int> q(n_req), kv(n_req);
        for (int r = 0; r < n_req; ++r) {
            q[r] = rnd(4) == 0 ? 0 : rnd(2) ? 1 + rnd(4) : 1 + rnd(900);
            kv[r] = rnd(5) == 0 ? rnd(q[r] + 1) : q[r] + rnd(3000);
        }
        for (int is_long = 0; is_long < 2; ++is_long) {
            long long total = 0;
            for (int r = 0; r < n_req; ++r) total += request_units(s, is_long, q[r], kv[r]);
            const int parts = 1 + rnd(300);
            CHECK(part_begin(total, 0, parts) == 0 && part_begin(total, parts, parts) == total);
            // the line, unit by unit
            long long at = 0;
            int part = 0;
            for (int r = 0; r < n_req; ++r) {
                CHECK(is_short(s, q[r]) == ((long long)q[r] * s.group <= kShortRows));
                const long long n = request_units(s, is_long, q[r], kv[r]);
                if (n == 0) continue;
                const int tiles = is_long ? long_tiles(s, q[r]) : 1;
                CHECK(!is_long || (tiles - 1) * s.tile < q[r]);
                CHECK(!is_long || tiles * s.tile >= q[r]);
                long long off = 0;
                for (int h = 0; h < s.n_kv; ++h)
                    for (int t = 0; t < tiles; ++t) {
                        const int units = is_long ? long_units(s, q[r], kv[r], t) : short_units(s, q[r], kv[r]);
                        const int last = is_long ? (t + 1) * s.tile < q[r] ? (t + 1) * s.tile - 1 : q[r] - 1 : q[r] - 1;
                        const int lim = row_limit(s, q[r], kv[r], last), u = is_long ? kLongUnit : s.unit;
                        CHECK(units >= 1 && (long long)units * u >= lim && (units == 1 || (units - 1) * u < (is_long ? lim : kv[r])));
                        for (int i = 0; i < units; ++i, ++off) {
                            const Place p = place_of(s, is_long, q[r], kv[r], off);
                            CHECK(p.head == h && p.tile == t && p.unit == i && p.units == units);
                        }
                    }
                CHECK(off == n);
                if (is_long) {
                    long long sum = 0;
                    for (int t = 0; t <= tiles; ++t) {
                        CHECK(long_units_before(s, q[r], kv[r], t) == sum);
                        if (t < tiles) sum += long_units(s, q[r], kv[r], t);
                    }
                }
                at += n;
            }
            CHECK(at == total);
            for (part = 0; part < parts; ++part) {
                const long long b = part_begin(total, part, parts), e = part_begin(total, part + 1, parts);
                CHECK(b <= e && e - b <= total / parts + 1);
            }
        }
    }
    // rows before position 0, lengths at their ends
    Shape s{4, 2, 64, 1, 64};
    CHECK(row_limit(s, 5, 2, 0) == 0 && row_limit(s, 5, 2, 4) == 2 && row_limit(s, 5, 2, 3) == 1);
    CHECK(row_limit(s, 1, 2147483647, 0) == 2147483647 && short_units(s, 1, 2147483647) == 33554432);
    CHECK(part_begin(1ll << 50, 511, 512) == (1ll << 50) / 512 * 511);
    CHECK(!lengths_ok(0, 5, 3, 4, 100) && !lengths_ok(3, 2, 3, 4, 100) && !lengths_ok(-1, 2, 3, 4, 100) && !lengths_ok(0, 1, 101, 4, 100) &&
          !lengths_ok(0, 1, -1, 4, 100) && lengths_ok(4, 4, 100, 4, 100));
    std::printf("ok\n");
    return 0;
}
