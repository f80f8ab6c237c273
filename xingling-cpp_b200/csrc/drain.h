// A draining warp's turn through a product's TMEM accumulators: waits for
// done[acc] (a K-block's sums are there), reads, and hands the accumulator
// back with an arrival on freed[acc].  Shared by the kernels and by the check
// that runs on the host.
#pragma once
#include <stdint.h>

#include "xl_hd.h"

namespace xl {

// `freed` is an array of 2 ACCS barriers; nobody waits for the second half.
template <int ACCS>
struct DrainTurn {
    static_assert((ACCS & (ACCS - 1)) == 0, "a power of two");
    int acc = 0;
    uint32_t parity = 0;  // of done[acc]
    bool ok = true;       // every wait so far ended in time
    // Arrivals are counted, not named: one by a warp that no longer waits would
    // complete the phase of another that still reads, and the next K-block
    // would be multiplied over what that one reads.  So a warp whose wait ran
    // out moves on to the half that nobody waits for; the issuing warp's wait
    // for it runs out in turn, and with that every other warp's, whose results
    // say so too.  (In acc itself, since the large product has no register to
    // spare: a branch around the arrival cost it 2.5 %, a second address 3.5 %.)
    XL_HD void waited(bool in_time) {
        ok = in_time;
        if (!in_time) acc += ACCS;
    }
    XL_HD void next() {
        acc ^= (acc ^ (acc + 1)) & (ACCS - 1);
        if ((acc & (ACCS - 1)) == 0) parity ^= 1u;
    }
};

}  // namespace xl
