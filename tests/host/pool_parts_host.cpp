// How many parts the line of kg_pool_attend_dev's work is cut into (kg_pool_sched.h), on the CPU: no part is empty, none
// begins or ends inside more than one item, few items get a part each, and long lines as many as there are CTAs.
#include <cstdio>
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
#define CHECK(x)                                        \
    do {                                                \
        if (!(x)) {                                     \
            std::printf("line %d: %s\n", __LINE__, #x); \
            return 1;                                   \
        }                                               \
    } while (0)

int main() {
    const int groups[] = {1, 2, 3, 4, 5, 7, 8, 16, 33, 64}, ctas[] = {296, 148, 1, 7};
    for (int trial = 0; trial < 4000; ++trial) {
        const int group = groups[rnd(10)];
        const Shape s{group, 1 + rnd(4), 2 * (128 / group), rnd(2), rnd(2) ? 64 : 128};
        const int n_req = 1 + rnd(12), most = ctas[rnd(4)], least = 2;
        std::vector<int> q(n_req), kv(n_req);
        for (int r = 0; r < n_req; ++r) {
            q[r] = rnd(4) == 0 ? 0 : rnd(2) ? 1 + rnd(4) : 1 + rnd(400);
            kv[r] = rnd(5) == 0 ? rnd(q[r] + 1) : rnd(8) ? q[r] + rnd(700) : q[r] + rnd(90000);
        }
        for (int is_long = 0; is_long < 2; ++is_long) {
            std::vector<long long> begin;  // of every item in the line, and its end
            long long total = 0, items = 0;
            for (int r = 0; r < n_req; ++r) {
                const long long here = request_items(s, is_long, q[r], kv[r]);
                items += here;
                const int tiles = is_long ? long_tiles(s, q[r]) : here > 0;
                CHECK(here == (long long)tiles * s.n_kv);
                CHECK((here == 0) == (request_units(s, is_long, q[r], kv[r]) == 0));
                for (int h = 0; h < s.n_kv; ++h)
                    for (int t = 0; t < tiles; ++t) {
                        begin.push_back(total);
                        total += is_long ? long_units(s, q[r], kv[r], t) : short_units(s, q[r], kv[r]);
                    }
            }
            begin.push_back(total);
            CHECK((long long)begin.size() == items + 1);
            const int parts = parts_of(total, items, most, least);
            CHECK(parts <= most && (total == 0) == (parts == 0));
            if (total == 0) continue;
            CHECK(parts <= total);
            CHECK(parts == most || parts >= items);  // an item each where they suffice
            CHECK(parts == most || parts * least >= total);
            CHECK(part_begin(total, 0, parts) == 0 && part_begin(total, parts, parts) == total);
            size_t at = 0;  // the item that holds the part's first unit
            for (int c = 0; c < parts; ++c) {
                const long long b = part_begin(total, c, parts), e = part_begin(total, c + 1, parts);
                CHECK(b < e);
                while (begin[at + 1] <= b) ++at;
                // cut items of the part: at most the one that holds its first unit (if it began before) and the one that
                // holds its last (if it ends behind), and of these at most one whose begin is here
                int open = 0, started = 0;
                for (size_t i = at; i + 1 < begin.size() && begin[i] < e; ++i) {
                    const bool before = begin[i] < b, behind = begin[i + 1] > e;
                    open += before;
                    started += !before && behind;
                }
                CHECK(open <= 1 && started <= 1);
            }
        }
    }
    CHECK(parts_of(0, 0, 296, 2) == 0 && parts_of(1, 1, 296, 2) == 1 && parts_of(40, 40, 296, 2) == 40 && parts_of(40, 1, 296, 2) == 20);
    CHECK(parts_of(1ll << 50, 1, 296, 2) == 296 && parts_of(1ll << 50, 1ll << 40, 296, 2) == 296);
    std::printf("ok\n");
    return 0;
}
