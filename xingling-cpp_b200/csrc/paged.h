// Where a paged key/value cache keeps a position and how attention over it is
// cut: arithmetic shared by the kernels and by the check that runs on the host.
#pragma once
#include <stdint.h>

#include "xl_hd.h"

namespace xl {

// n / d for 0 <= n < 2^31 with a multiplication (Granlund and Montgomery,
// "Division by invariant integers using multiplication", PLDI 1994): with
// l = ceil(log2 d) and mul = floor(2^32 (2^l - d) / d) + 1 the quotient is
// (hi + (n - hi) / 2) >> (l - 1), hi the high word of n * mul.
struct FastDiv {
    uint32_t d, mul, shift;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        uint32_t l = 0;
        while ((1ull << l) < div) ++l;
        mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << l) - div)) / div + 1);
        shift = l;
    }
    XL_HD uint32_t div(uint32_t n) const {
#ifdef __CUDA_ARCH__
        const uint32_t hi = __umulhi(n, mul);
#else
        const uint32_t hi = static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> 32);
#endif
        return shift ? (hi + ((n - hi) >> 1)) >> (shift - 1) : n;
    }
};

// A pool of pages [num_pages][kv_heads][page_size][head_dim] for keys and one
// for values; page_table [batch][max_pages] names the pages of each sequence.
struct PagedCache {
    void* k;
    void* v;
    const int* page_table;
    int dtype;
    int batch, kv_heads, head_dim, page_size, max_pages, num_pages;
};

// Element offset of (page, head, slot 0) in a pool, 64-bit: a pool may hold more than 2^31 elements.
XL_HD int64_t paged_base(int page, int head, int kv_heads, int page_size, int head_dim) {
    return (static_cast<int64_t>(page) * kv_heads + head) * page_size * head_dim;
}
XL_HD bool paged_valid(int page, int num_pages) { return page >= 0 && page < num_pages; }

// Whether position pos of a sequence can be held at all: -1 (a slot without a
// sequence) is told apart by the callers.
XL_HD bool paged_pos_ok(int pos, int max_pages, int page_size, int rope_len) {
    return pos >= 0 && pos < static_cast<int64_t>(max_pages) * page_size && (rope_len == 0 || pos < rope_len);
}

// Attention's work: `all` units in a row, cut over `grid` CTAs (grid <= all),
// CTA i taking [paged_share(i), paged_share(i + 1)); paged_owner is the CTA
// that takes a unit.  64-bit divisions take hundreds of clocks on the device:
// 32 bits where all * (grid + 1) fits (`brief`).
constexpr int kPagedMaxCtas = 740;  // 148 SMs x 5
XL_HD bool paged_brief(int64_t all) { return all < (static_cast<int64_t>(1) << 31) / (kPagedMaxCtas + 1); }
XL_HD int64_t paged_share(uint32_t i, int64_t all, int64_t grid, bool brief) {
    return brief ? static_cast<int64_t>(i * static_cast<uint32_t>(all) / static_cast<uint32_t>(grid)) : i * all / grid;
}
XL_HD int paged_owner(int64_t unit, int64_t all, int64_t grid, bool brief) {
    const int64_t v = (unit + 1) * grid - 1;
    return brief ? static_cast<int>(static_cast<uint32_t>(v) / static_cast<uint32_t>(all)) : static_cast<int>(v / all);
}

}  // namespace xl
