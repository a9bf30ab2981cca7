// The ring of stages of kg_pool_attend_dev's kernels (kg_pool_ring.h) on host threads, with barriers that count as the
// device's do and waits that run out at random: the lanes of a warp have to go on alike, no stage is filled again while a
// load into it is under way, no load is left when the loader ends, and everyone ends.
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

// ---- the lanes of one warp
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

// ---- a loader, its copies, and the warps that use the stages
struct Barrier {  // counts arrivals and bytes; a phase ends when neither is missing
    std::mutex mu;
    int expected = 0, pending = 0, phase = 0;
    long bytes = 0;
    void init(int n) { expected = pending = n; }
    void step() {
        if (pending == 0 && bytes == 0) {
            ++phase;
            pending = expected;
        }
    }
    void arrive(long more = 0) {
        std::lock_guard<std::mutex> lk(mu);
        CHECK(pending > 0);  // the phase before has not ended
        bytes += more;
        --pending;
        step();
    }
    void arrived(long n) {
        std::lock_guard<std::mutex> lk(mu);
        bytes -= n;
        step();
    }
    bool done(int parity) {
        std::lock_guard<std::mutex> lk(mu);
        return (phase & 1) != parity;
    }
};

constexpr int STAGES = 6, USERS = 4, BYTES = 100;

struct Block {
    Barrier full[STAGES], empty[STAGES];
    int stage[STAGES];                 // the load that it holds
    std::atomic<int> abort_flag{0};
    std::mutex mu;
    std::vector<int> under_way;        // loads
    std::atomic<int> left{0}, gone{0};  // loads under way, copies to be ended
    Vote vote[USERS];
};

struct Thread {  // the barriers as one thread sees them; `fail`: one wait of so many runs out (0: none)
    Block &k;
    unsigned seed;
    int fail, user;
    bool wait(Barrier &b, int parity) {
        if (b.done(parity)) return true;
        const bool out = fail && rnd(seed, fail) == 0;
        for (int tries = 0; !b.done(parity); ++tries) {
            if (k.abort_flag) return false;
            if (out && tries > 3) {
                k.abort_flag = 1;
                return false;
            }
            std::this_thread::yield();
        }
        return true;
    }
    bool wait_full(int s, int parity) { return wait(k.full[s], parity); }
    bool wait_empty(int s, int parity) { return wait(k.empty[s], parity); }
    void arm(int s) { k.full[s].arrive(BYTES); }
    void free(int s) { k.empty[s].arrive(); }
    bool all(bool x) { return k.vote[user].all(x); }
    void landed(int s, int parity) {
        while (!k.full[s].done(parity)) std::this_thread::yield();
    }
};

static void block(unsigned seed, int stages, int loads, int fail) {
    Block k;
    for (int i = 0; i < stages; ++i) {
        k.full[i].init(1);
        k.empty[i].init(USERS);
    }
    std::thread copies([&] {  // loads end late, in any order
        unsigned r = seed * 7919u + 1;
        const unsigned slow = seed % 2 ? 3 : 300;
        while (!k.gone || k.left) {
            int it = -1;
            {
                std::lock_guard<std::mutex> lk(k.mu);
                if (!k.under_way.empty() && rnd(r, slow) == 0) {
                    const size_t i = rnd(r, k.under_way.size());
                    it = k.under_way[i];
                    k.under_way.erase(k.under_way.begin() + i);
                }
            }
            if (it < 0) {
                std::this_thread::yield();
                continue;
            }
            k.stage[it % stages] = it;
            --k.left;
            k.full[it % stages].arrived(BYTES);
        }
    });
    std::vector<std::thread> threads;
    threads.emplace_back([&] {
        Thread b{k, seed * 31u + 5, fail, 0};
        int it = 0;
        for (; it < loads; ++it) {
            if (!ring_claim(b, stages, it)) break;
            ++k.left;
            std::lock_guard<std::mutex> lk(k.mu);
            k.under_way.push_back(it);
        }
        CHECK(fail || it == loads);
        ring_drain(b, stages, it);
        CHECK(k.left == 0);
        k.gone = 1;
    });
    std::atomic<int> saw[USERS][LANES];
    for (int w = 0; w < USERS; ++w)
        for (int l = 0; l < LANES; ++l)
            threads.emplace_back([&, w, l] {
                Thread b{k, seed * 131u + w * 17 + l + 3, fail, w};
                bool alive = true;
                for (int it = 0; it < loads; ++it) {
                    alive = ring_take(b, stages, it, alive);
                    if (alive) CHECK(k.stage[it % stages] == it);
                    saw[w][l] = alive;
                    b.all(true);  // (the lanes have used the stage)
                    if (l == 0) {
                        CHECK(saw[w][0] == saw[w][1]);
                        ring_free(b, stages, it, alive);
                    }
                    b.all(true);
                }
                CHECK(fail || alive);
            });
    for (auto &t : threads) t.join();
    copies.join();
}

int main() {
    for (unsigned i = 1; i <= 300 && !bad; ++i) lanes_agree(i);
    for (unsigned i = 1; i <= 1500 && !bad; ++i) block(i, i % 7 == 0 ? 1 : i % 2 ? 3 : 4 + i % 3, 1 + i % 23, i % 5 == 0 ? 0 : i % 3 == 0 ? 2 : 12);
    if (!bad) std::printf("ok\n");
    return bad != 0;
}
