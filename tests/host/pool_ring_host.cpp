// The ring of stages of kg_pool_attend_dev's kernels (kg_pool_ring.h) on host threads, with barriers that count as the
// device's do and waits that run out at random: the lanes of a warp have to go on alike.
#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <thread>
#include <vector>

#include "../../katgpt-rs_b200/csrc/kg_pool_ring.h"

using namespace kg::serve;

static std::atomic<int> bad{0};
#define CHECK(x)                                                        \
    do {                                                                \
        if (!(x) && bad++ == 0) std::printf("line %d: %s\n", __LINE__, #x); \
    } while (0)

static unsigned rnd(unsigned &s, unsigned n) {
    s ^= s << 13;
    s ^= s >> 17;
    s ^= s << 5;
    return s % n;
}

constexpr int LANES = 2;

// a point where the lanes of a warp meet: all of their votes
struct Vote {
    std::atomic<int> count{0}, turn{0}, no[2] = {{0}, {0}};
    bool all(bool x) {
        const int t = turn.load();
        if (!x) no[t & 1] = 1;
        if (++count == LANES) {
            no[(t + 1) & 1] = 0;
            count = 0;
            ++turn;
        } else {
            while (turn.load() == t) std::this_thread::yield();
        }
        return no[t & 1] == 0;
    }
};

struct Lane {
    Vote &vote;
    unsigned seed;
    int fail;  // one wait of so many runs out
    bool wait_full(int, int) { return rnd(seed, fail) != 0; }
    bool all(bool x) { return vote.all(x); }
};

static void lanes_agree(unsigned seed) {
    constexpr int N = 40;
    Vote vote;
    char saw[LANES][N];
    std::vector<std::thread> threads;
    for (int l = 0; l < LANES; ++l)
        threads.emplace_back([&, l] {
            Lane b{vote, seed * 2654435761u + l * 97 + 1, 20};
            bool alive = true;
            for (int it = 0; it < N; ++it) saw[l][it] = alive = ring_take(b, 3, it, alive);
        });
    for (auto &t : threads) t.join();
    for (int it = 0; it < N; ++it) {
        CHECK(saw[0][it] == saw[1][it]);
        CHECK(it == 0 || saw[0][it] <= saw[0][it - 1]);
    }
}

int main() {
    for (unsigned i = 1; i <= 300 && !bad; ++i) lanes_agree(i);
    if (!bad) std::printf("ok\n");
    return bad != 0;
}
