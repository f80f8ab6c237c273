// Host-side check of drain.h: warps drain accumulators that one issuer fills,
// in random orders of their steps, one warp's wait running out at a random
// K-block.  Whatever a warp reads after a wait that ended in time has to be its
// K-block's sums.  Prints "ok", or the first failure.
#include <cstdio>
#include <random>
#include <vector>

#include "drain.h"

using namespace xl;

// An mbarrier as waits by parity see it: waiting on a parity ends when the phase under way has the other one.
struct Barrier {
    int count, pending, phase = 0;
    explicit Barrier(int n) : count(n), pending(n) {}
    void arrive() {
        if (--pending == 0) pending = count, ++phase;
    }
    bool passed(uint32_t parity) const { return (static_cast<uint32_t>(phase) & 1u) != parity; }
};

template <int ACCS>
bool run(std::mt19937& rng, int warps, int blocks, int late_warp, int late_block) {
    std::vector<Barrier> done(ACCS, Barrier(1)), freed(2 * ACCS, Barrier(warps));
    int held[ACCS];  // the K-block whose sums an accumulator holds
    struct Warp {
        DrainTurn<ACCS> turn;
        int block = 0, step = 0;
    };
    std::vector<Warp> w(warps);
    int issued = 0, acc = 0, idle = 0;
    uint32_t parity = 0;
    bool issue_step = false;
    while (idle < 1000) {  // until no wait ends any more (the kernel's run out then)
        const int who = static_cast<int>(rng() % (warps + 1));
        ++idle;
        if (who == warps) {
            if (issued == blocks) continue;
            if (!issue_step) {
                issue_step = freed[acc].passed(parity ^ 1u);
                if (issue_step) idle = 0;
                continue;
            }
            held[acc] = issued++, done[acc].arrive(), issue_step = false, idle = 0;
            if (++acc == ACCS) acc = 0, parity ^= 1u;
            continue;
        }
        Warp& a = w[who];
        if (a.block == blocks) continue;
        if (a.step == 0) {  // the wait
            if (a.turn.ok && who == late_warp && a.block == late_block)
                a.turn.waited(false);
            else if (a.turn.ok && !done[a.turn.acc].passed(a.turn.parity))
                continue;
        } else if (a.step == 1) {  // the reads
            if (a.turn.ok && held[a.turn.acc] != a.block) {
                std::printf("warp %d read K-block %d where it waited for %d\n", who, held[a.turn.acc], a.block);
                return false;
            }
        } else {
            freed[a.turn.acc].arrive();
            a.turn.next();
            ++a.block;
        }
        a.step = (a.step + 1) % 3;
        idle = 0;
    }
    if (late_warp >= 0) return true;
    for (const Warp& a : w)
        if (a.block != blocks) {
            std::printf("a warp stopped at %d of %d\n", a.block, blocks);
            return false;
        }
    return true;
}

int main() {
    std::mt19937 rng(1);
    for (int i = 0; i < 2000; ++i) {
        const int warps = i % 2 ? 4 : 16, blocks = 1 + static_cast<int>(rng() % 40);
        const int late = i % 5 ? static_cast<int>(rng() % warps) : -1, at = static_cast<int>(rng() % blocks);
        if (!run<2>(rng, warps, blocks, late, at) || !run<4>(rng, warps, blocks, late, at) || !run<8>(rng, warps, blocks, late, at))
            return 1;
    }
    std::printf("ok\n");
    return 0;
}
