// Where a paged key/value cache keeps a position: arithmetic shared by the
// kernels and by the host-side check that runs without a GPU.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define XL_HD __host__ __device__ __forceinline__
#else
#define XL_HD inline
#endif

namespace xl {

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

}  // namespace xl
