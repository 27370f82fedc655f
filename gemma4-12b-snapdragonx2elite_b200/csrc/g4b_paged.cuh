// g4b_paged.cuh -- what the paged-cache kernels share: the plan of a ragged batch, its layout in the
// caller's buffer, the walk over its pieces, and where a piece's partial result goes.
//
// A batch is B sequences with their new tokens back to back in rows [q_start[b], q_start[b + 1]) of the
// token buffers.  Sequence b holds kv_len[b] tokens once its new ones are appended; its token i has
// position kv_len[b] - n_b + i.  Positions below prefix_len live in the pages of one prefix table that all
// sequences share, the others in the sequence's own table row.
//
// The attention of a KV head is cut into tiles: rows (row = token * G + query head of the group) against keys, in
// units of 64 keys.  A sequence with up to few_most rows (a decode step, a few proposed tokens) has a tile of its own keys
// for the few-rows kernel (or two, of kRowsS rows each), one with more has tiles of kRowsP rows.  Up to kRowsAlone, its rows also join those of
// the other such sequences in tiles against the prefix; with more (a prompt's chunk) it fills tiles by itself,
// which read the prefix and then its own keys.  The units of all tiles and KV heads
// form one line that is cut into equal lengths, one per CTA, whatever the lengths of the sequences: a CTA
// walks its stretch piece by piece.  (A tile counts for a few units more than it has: its start and end take time too.)
// Where that costs no more (few tiles, many CTAs) every tile starts at a border.  A tile that lies in one CTA's stretch is finished there; one that
// crosses a border leaves a partial (running maximum, sum, weighted values) in the edge slots of each CTA,
// and the join kernel adds them.
#pragma once

#include "g4b_common.cuh"
#include "g4b_pages.h"

namespace g4b {
namespace pg {

constexpr int kUnit = 64;        // keys per unit of work
constexpr int kRowsS = 8;        // rows of a tile of the few-rows kernel (the n of m16n8k16)
// A sequence of up to this many rows goes to the few-rows kernel, in one tile or two.  Two tiles read the keys twice,
// mostly from L2: at hd 128 that is faster than a 128-row tile with 16 rows in it (64 sequences of 16 rows over 2,000
// keys: 31 us against 40; over 200: 12 against 17), from hd 256 on only for short sequences (32 of 16 rows over
// 2,000 keys: 174 us against 122).
constexpr int few_most(int hd) { return hd == 128 ? 16 : 8; }
constexpr int kRowsP = 128;      // rows of a tile of the many-rows kernel (tensor memory lanes)
// A sequence of more rows than this reads the prefix in its own tiles; one of fewer shares tiles of the prefix with
// others and has its partial results joined.  Half a tile: by itself it would use less of a tile's products than that.
constexpr int kRowsAlone = 64;
constexpr int kMaxSeqs = 4096;   // the plan kernel keeps the sequences in shared memory
constexpr unsigned kStatusPlan = 2u;   // a plan made for other sizes (or never made) was passed

struct __align__(16) Tile {
    int row0;        // first row: token * G + g
    int nrows;       // rows of the tile
    int seq;         // sequence whose own keys it reads; -1: the shared prefix alone
    int n;           // units: first n1 of the prefix, then the sequence's own
    int n1, lo1, hi1;   // prefix keys [lo1, hi1); lo1 is a multiple of kUnit
    int lo2, hi2;       // own keys [lo2, hi2), counted from the prefix's end; lo2 is a multiple of kUnit
    int solo;        // its rows have keys in no other tile: a whole tile writes the output itself
    int idle;        // units behind it that are nobody's work: what the tile costs besides its units, or what aligns the
                     // next one with a stretch's start
    int pad;
    long long off;   // units of the tiles before it, their idle ones included
    long long pad2;
};

// unit u of a tile: its first key (in the prefix's or the sequence's own count), its segment, the segment's end
struct Unit {
    bool pre;
    int key, hi;
};
__host__ __device__ __forceinline__ Unit unit_of(const Tile& t, int u) {
    const bool pre = u < t.n1;
    return {pre, pre ? t.lo1 + u * kUnit : t.lo2 + (u - t.n1) * kUnit, pre ? t.hi1 : t.hi2};
}

struct Start {       // where a CTA's stretch begins
    int head, tile, unit;        // head: KV head * walks per tile + walk; -1: nothing to do
    int skip;                    // idle units before that
    Tile t;                      // tiles[tile]
};

struct Hdr {
    PlanKey key;                     // the sizes the plan was made for
    int prefix_len;
    int tok_lo, tok_hi;              // rows of the token buffers that belong to a sequence
    int nt[2];                       // tiles: [0] few rows, [1] many rows
    int nj[2];                       // entries of the join kernel's lists,
    int rj[2];                       // and the rows that one stands for
    long long wt[2];                 // units of one KV head
    long long u[2];                  // units per CTA
};

// sizes fixed on the host, and the offsets of the arrays in the plan buffer that follow from them
struct Dims {
    int T, B, nH, nkv, G, hd, ps, own_pages, pre_pages, window;
    int lps;                         // log2 of the page size
    int few;                         // few_most(hd)
    int cs;                          // walks per many-rows tile: parts of hd's output columns
    int ctas[2];                     // stretches per kind
    int max_tiles[2];
    int join_ctas;                   // CTAs of the join kernel that are there at once
    size_t tok_seq, tok_pos, row_pre, start[2], tiles[2], joins[2], bytes;
    PlanKey key;
};

__host__ __device__ inline const Hdr* hdr_of(const void* plan) { return reinterpret_cast<const Hdr*>(plan); }
template <typename X>
__host__ __device__ inline X* at(void* plan, size_t off) {
    return reinterpret_cast<X*>(reinterpret_cast<char*>(plan) + off);
}
template <typename X>
__host__ __device__ inline const X* at(const void* plan, size_t off) {
    return reinterpret_cast<const X*>(reinterpret_cast<const char*>(plan) + off);
}

// The plan is one that was made for this call's sizes: all its offsets and row numbers are taken from it.
__device__ __forceinline__ bool plan_fits(const Hdr* h, const Dims& d) { return same_plan(h->key, d.key); }

// The workspace: edge slots of both kinds ([cta][2][rows][columns of a walk] sums, [cta][2][rows] (max, sum)), then,
// where there is a prefix, one slot per (segment kind, token, head) for whole tiles.
struct Work {
    float* edge[2];
    float2* edge_ml[2];
    float* row;        // [2][T * nH][hd]: 0 prefix, 1 own
    float2* row_ml;    // [2][T * nH][2]: one per walk of the tile (the few-rows kernel's only one first)
};

struct Args {
    const void* plan;
    const uint16_t* q;
    const uint16_t* kc;
    const uint16_t* vc;
    const int* table;
    const int* pre_table;
    void* out;
    Work w;
    long long q_stride, out_stride;
    float scale;       // times log2(e): scores are kept in powers of two
    int out_f32, num_pages;
    Dims d;
};

__device__ __forceinline__ Span span_of(const Hdr* h, int kind, long long off, int n, int head) {
    return span_of((long long)head * h->wt[kind] + off, n, h->u[kind]);
}

// mbar_wait whose first tries do not read the timer: in these kernels most waits are short and lie on the path
// from one unit to the next.
__device__ __forceinline__ bool wait_short(uint32_t bar, uint32_t parity, volatile int* abort, unsigned* status) {
    #pragma unroll 1
    for (int i = 0; i < 64; i++)
        if (mbar_try_wait(bar, parity)) return true;
    return mbar_wait(bar, parity, abort, status);
}

// The same for a whole warp in little code, without the timer (the many-rows kernel is 4 % faster for it).  Bounded by its
// tries: each takes 40 clocks (0.08 s in all) to as long as the hardware holds a warp back.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort, unsigned* status) {
    #pragma unroll 1
    for (int i = 0; i < 1 << 22; i++) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if ((i & 255) == 255 && __any_sync(0xffffffffu, *abort)) return false;
    }
    *abort = 1;
    atomicOr(status, kStatusTimeout);
    return false;
}

// a box of a tensor_map_chunks map: rows from `row`, 64-element chunks from `chunk`
__device__ __forceinline__ void tma_chunks(uint32_t dst, const CUtensorMap* map, int row, int chunk, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(chunk), "r"(bar)
        : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two f32 rounded to f16 by one instruction: the conversion of one at a time has a quarter of the rate.
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    const __half2 h2 = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h2);
}

// the many-rows kernel (g4b_paged_mma.cu): its launch, its status word
int launch_many(const Args& a, cudaStream_t s);
unsigned read_status_paged_mma();

}  // namespace pg
}  // namespace g4b
