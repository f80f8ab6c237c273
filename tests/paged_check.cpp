// Host-side check of paged.h: where a paged cache keeps a position, which
// positions and pages are refused, the division by multiplication, and how
// attention's work is cut over CTAs.  Prints "ok", or the first failure.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "paged.h"

using namespace xl;

#define CHECK(c)                                             \
    do {                                                     \
        if (!(c)) {                                          \
            std::printf("line %d: %s\n", __LINE__, #c);      \
            return 1;                                        \
        }                                                    \
    } while (0)

int main() {
    std::mt19937_64 rng(1);
    // pages and positions
    CHECK(!paged_valid(-1, 4) && !paged_valid(4, 4) && !paged_valid(1 << 30, 4) && paged_valid(0, 4) && paged_valid(3, 4));
    CHECK(!paged_pos_ok(-1, 4, 16, 0) && !paged_pos_ok(64, 4, 16, 0) && paged_pos_ok(63, 4, 16, 0) && paged_pos_ok(0, 4, 16, 0));
    CHECK(!paged_pos_ok(10, 4, 16, 10) && paged_pos_ok(9, 4, 16, 10) && !paged_pos_ok(-2147483647 - 1, 4, 16, 0));
    CHECK(paged_pos_ok(2147418111, 32767, 65536, 0) && !paged_pos_ok(2147418112, 32767, 65536, 0));
    CHECK(paged_base(3000000, 1, 8, 64, 128) == (3000000ll * 8 + 1) * 64 * 128);
    // division
    std::vector<uint32_t> divisors{1, 2, 3, 5, 7, 8, 12, 13, 16, 24, 100, 128, 1000, 65535, 65536, 65537, 1u << 30, 2147483647u};
    for (int i = 0; i < 300; ++i) divisors.push_back(1 + static_cast<uint32_t>(rng() % 2147483647u));
    for (uint32_t d : divisors) {
        const FastDiv f(d);
        std::vector<uint32_t> ns{0, 1, 2, d - 1, d, d + 1, 2147483646u, 2147483647u};
        for (int i = 0; i < 200; ++i) ns.push_back(static_cast<uint32_t>(rng() % 2147483648u));
        for (uint32_t k = 1; k < 50; ++k)
            if (static_cast<uint64_t>(k) * d < 2147483648ull) ns.push_back(k * d), ns.push_back(k * d - 1);
        for (uint32_t n : ns)
            if (n < 2147483648u) CHECK(f.div(n) == n / d);
    }
    // the cut: every unit belongs to one CTA, the one paged_owner names; every CTA has a unit; both divisions agree
    std::vector<int64_t> alls{1, 2, 3, 100, 443, 444, 445, 740, 741, 1000, 12345, 2897000, 2898000, 3000000, 1ll << 33, 1ll << 40};
    for (int64_t all : alls)
        for (int64_t most : {1, 7, 296, 444, 740}) {
            const int64_t grid = most < all ? most : all;
            const bool brief = paged_brief(all);
            CHECK(paged_share(0, all, grid, brief) == 0 && paged_share(static_cast<uint32_t>(grid), all, grid, brief) == all);
            for (int64_t i = 0; i < grid; ++i) {
                const int64_t a = paged_share(static_cast<uint32_t>(i), all, grid, brief);
                const int64_t b = paged_share(static_cast<uint32_t>(i + 1), all, grid, brief);
                CHECK(a < b && a == paged_share(static_cast<uint32_t>(i), all, grid, false));
                for (int64_t u : {a, (a + b) / 2, b - 1}) {
                    CHECK(paged_owner(u, all, grid, brief) == i);
                    CHECK(paged_owner(u, all, grid, false) == i);
                }
            }
        }
    std::printf("ok\n");
    return 0;
}
