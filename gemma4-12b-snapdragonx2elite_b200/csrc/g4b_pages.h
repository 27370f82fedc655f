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

// What a plan was made for: a call takes it only where every one of these is its own.  The first word is no size, so that
// memory of zeros, or of anything else, is not taken for a plan.
struct alignas(16) PlanKey {
    int v[12];       // magic, T, B, nH, nkv, hd, page_size, table_pages, prefix_pages, window, CTAs per kind
};
constexpr int kPlanMagic = 0x67346270;

G4B_HD bool same_plan(const PlanKey& a, const PlanKey& b) {
    int diff = 0;
    for (int i = 0; i < 12; i++) diff |= a.v[i] ^ b.v[i];
    return diff == 0;
}

// The CTAs whose stretches of `u` units hold the units [g, g + n) of the line of all work (n >= 1).
struct Span {
    int c0, c1;
};
G4B_HD Span span_of(long long g, int n, long long u) { return {(int)(g / u), (int)((g + n - 1) / u)}; }

}  // namespace pg
}  // namespace g4b
