// g4b_pages.h -- the paged cache's addressing, plain C++ so that the host can run it too.
#pragma once

#ifdef __CUDACC__
#define G4B_HD __host__ __device__ __forceinline__
#else
#define G4B_HD inline
#endif

namespace g4b {
namespace pg {

// Row of the cache, seen as [num_pages * nkv * page_size] rows of hd, that holds key `key` of a segment for KV
// head `head`, given the page's id and the log2 of the page size; -1 where the id names no page.
// num_pages * nkv * page_size < 2^31.
G4B_HD int cache_row(int page, int num_pages, int nkv, int log2_page_size, int head, int key) {
    if (page < 0 || page >= num_pages) return -1;
    return ((page * nkv + head) << log2_page_size) + (key & ((1 << log2_page_size) - 1));
}

// The CTAs whose stretches of `u` units hold the units [g, g + n) of the line of all work (n >= 1).
struct Span {
    int c0, c1;
};
G4B_HD Span span_of(long long g, int n, long long u) { return {(int)(g / u), (int)((g + n - 1) / u)}; }

}  // namespace pg
}  // namespace g4b
