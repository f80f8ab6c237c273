// Host-side check of per_device.h: each device's own answer, asked once.
// Prints "ok", or the first failure.
#include <cstdio>

#include "per_device.h"

#define CHECK(c)                                             \
    do {                                                     \
        if (!(c)) {                                          \
            std::printf("line %d: %s\n", __LINE__, #c);      \
            return 1;                                        \
        }                                                    \
    } while (0)

int main() {
    xl::PerDevice p;
    int asked = 0;
    auto get = [&](int device, int answer) { return p.get(device, [&] { return ++asked, answer; }); };
    CHECK(get(0, 36) == 36 && asked == 1);
    CHECK(get(1, 18) == 18 && asked == 2);  // not the first one's
    CHECK(get(0, 99) == 36 && get(1, 99) == 18 && asked == 2);
    CHECK(get(2, 0) == 0 && get(2, 7) == 7 && asked == 4);  // a failure is not kept
    CHECK(get(63, 5) == 5 && get(63, 6) == 5 && asked == 5);
    CHECK(get(64, 5) == 5 && get(64, 6) == 6 && get(1000, 1) == 1 && get(-1, 2) == 2 && asked == 9);  // nor further devices
    std::printf("ok\n");
    return 0;
}
