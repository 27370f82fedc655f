// g4b_paged.cu -- a batch of sequences over a paged f16 KV cache: the plan of the batch, the append of its new
// keys and values with norm and rotation, and its attention, with a prefix that all sequences share read for many of
// their rows at a time.
//
// The cache is [num_pages, nkv, page_size, hd] f16: the engine's per-head cache rows (src/vk_engine.py:281-282)
// cut into pages.  The arithmetic per token and head is that of vk/prepkv.comp and vk/attn.comp.
#include <algorithm>

#include "g4b_paged.cuh"
#include "g4b_tcgen05.cuh"   // mbar_wait_drain

namespace g4b {
namespace pg {

constexpr float kEps = 1e-6f;    // vk/attn.comp:25, vk/prepkv.comp:21
__device__ unsigned g_status_paged;

// ------------------------------------------------------------------ sizes
static size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// CTAs of the few-rows kernel per SM: two where the stages of two fit an SM's shared memory (hd 128, 256)
static int few_per_sm(int hd) { return hd == 512 ? 1 : 2; }

// The join kernel's warps per CTA, and its CTAs per SM.  They are there early and wait: with four or eight an SM, 64 users
// of a long prefix take 101 and 107 us instead of 100, 128 users at hd 128 29 and 32 instead of 27; with one, chunks
// under a window 214 instead of 196.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kJoinPerSm = 2;

// Checks the sizes and lays the plan out for `sms` SMs.  No device is needed: a caller that will launch asks
// check_device() last, when every argument has been looked at.
static int make_dims(const char* op, int T, int B, int nH, int nkv, int hd, int ps, int own_pages, int pre_pages,
                     int window, Dims& d) {
    G4B_REQUIRE(T >= 1 && B >= 1 && B <= kMaxSeqs, G4B_E_SHAPE, "%s: T=%d tokens, B=%d sequences (1 to %d)", op, T, B,
                kMaxSeqs);
    G4B_REQUIRE(nkv >= 1 && nkv <= 65535 && nH <= 262144 && nH >= nkv && nH % nkv == 0 && (hd == 128 || hd == 256 || hd == 512),
                G4B_E_SHAPE, "%s: nH=%d nkv=%d hd=%d (nH a multiple of nkv, hd 128, 256 or 512)", op, nH, nkv, hd);
    G4B_REQUIRE(ps >= 16 && ps <= 1024 && (ps & (ps - 1)) == 0, G4B_E_SHAPE,
                "%s: page_size=%d (a power of two from 16 to 1024)", op, ps);
    G4B_REQUIRE(own_pages >= 1 && pre_pages >= 0 && window >= 0 &&
                    ((long long)own_pages + pre_pages) * ps <= 0x40000000LL,
                G4B_E_SHAPE, "%s: table of %d pages, prefix of %d, page_size %d, window %d (at most 2^30 positions)",
                op, own_pages, pre_pages, ps, window);
    G4B_REQUIRE((long long)T * nH <= 0x20000000LL, G4B_E_SHAPE, "%s: T=%d tokens of %d heads are too many", op, T, nH);
    int sms = 148;
    if (check_device(&sms) != G4B_OK) sms = 148;
    clear_error();
    d = Dims{};
    d.T = T;
    d.B = B;
    d.nH = nH;
    d.nkv = nkv;
    d.G = nH / nkv;
    d.hd = hd;
    d.ps = ps;
    d.own_pages = own_pages;
    d.pre_pages = pre_pages;
    d.window = window < 0x40000000 ? window : 0;     // no position is as far as that from another
    while ((1 << d.lps) < ps) d.lps++;
    d.few = few_most(hd);
    d.cs = hd == 512 ? 2 : 1;
    d.ctas[0] = sms * few_per_sm(hd);
    d.ctas[1] = sms;
    d.join_ctas = sms * kJoinPerSm;
    const int rows = T * d.G;
    // tiles of sequences (one more each for the last, partial one) and of the prefix
    d.max_tiles[0] = (B + 1) * (d.few / kRowsS);
    d.max_tiles[1] = 2 * (rows / kRowsP) + B + 1;
    size_t o = up256(sizeof(Hdr));
    auto take = [&](size_t bytes) {
        const size_t at = o;
        o += up256(bytes);
        return at;
    };
    d.tok_seq = take((size_t)T * 4);
    d.tok_pos = take((size_t)T * 4);
    d.row_pre = take((size_t)rows * 4);
    for (int k = 0; k < 2; k++) {
        d.start[k] = take((size_t)d.ctas[k] * sizeof(Start));
        d.tiles[k] = take((size_t)d.max_tiles[k] * sizeof(Tile));
        // a list has an entry per group of eight rows, or at most join_ctas smaller ones
        d.joins[k] = take(std::max((size_t)d.max_tiles[k] * nkv * ((k ? kRowsP : kRowsS) / kJoinWarps), (size_t)d.join_ctas) * sizeof(int2));
    }
    d.bytes = o;
    d.key = {{kPlanMagic, T, B, nH, nkv, hd, ps, own_pages, pre_pages, d.window, d.ctas[0], d.ctas[1]}};
    return G4B_OK;
}

static size_t work_bytes(const Dims& d, char* base, Work* w) {
    size_t o = 0;
    auto take = [&](size_t bytes) {
        const size_t at = o;
        o += up256(bytes);
        return base + at;
    };
    Work x{};
    for (int k = 0; k < 2; k++) {
        const size_t rows = (size_t)d.ctas[k] * 2 * (k ? kRowsP : kRowsS);
        x.edge[k] = reinterpret_cast<float*>(take(rows * (k ? d.hd / d.cs : d.hd) * 4));
        x.edge_ml[k] = reinterpret_cast<float2*>(take(rows * 8));
    }
    if (d.pre_pages > 0) {
        const size_t rows = (size_t)d.T * d.nH * 2;
        x.row = reinterpret_cast<float*>(take(rows * d.hd * 4));
        x.row_ml = reinterpret_cast<float2*>(take(rows * 2 * 8));
    }
    if (w) *w = x;
    return o;
}

// ------------------------------------------------------------------ plan
// Every CTA reads the sequences into shared memory and makes its share of the per-token and per-row
// arrays; CTA 0 makes the tiles, whose offsets are one running sum.  Nothing the caller's lengths say is
// trusted with an address: starts are made non-decreasing and cut to [0, T], lengths to the tables'
// capacity.
constexpr int kPlanThreads = 1024;
// A tile's start and end cost about as much as this many of its units (rows in, masks, result out): they count as its
// work, or a causal prompt's short first tiles, twenty to a stretch, make the slowest CTA (2 prompts of 4,096: with none
// 369 us at hd 256 and 221 at hd 128, with 5 units 310 and 125, with 8 to 10 293 and 122; ragged decode, 48 tokens: with
// none 143 us, with 2 units 140).  A border inside a tile costs its CTA another start and another partial.
constexpr int kTileCostS = 2, kTileCostP = 8, kBorderCostS = 2, kBorderCostP = 3;

struct PlanArgs {
    const int* q_start;
    const int* kv_len;
    const int* prefix_len;
    void* plan;
    Dims d;
};

__device__ __forceinline__ int seq_of(const int* st, int B, int t) {   // the last b with st[b] <= t
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (st[m] <= t) lo = m;
        else hi = m;
    }
    return lo;
}

template <typename X, typename F>
__device__ X block_scan(X v, X init, X* warp_buf, X* total, F op) {   // exclusive; total: of the whole block
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    X inc = v;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const X u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc = op(u, inc);
    }
    X exc = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 0) exc = init;
    __syncthreads();
    if (lane == 31) warp_buf[warp] = inc;
    __syncthreads();
    X before = init, all = init;
    for (int w = 0; w < kPlanThreads / 32; w++) {
        if (w == warp) before = all;
        all = op(all, warp_buf[w]);
    }
    *total = all;
    return op(before, exc);
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
    extern __shared__ int sm[];
    __shared__ long long wbuf[kPlanThreads / 32];
    __shared__ int ibuf[kPlanThreads / 32], s_joins, s_rows[4];
    const Dims& d = a.d;
    const int B = d.B, G = d.G, tid = threadIdx.x;
    int* st = sm;                    // [B + 1] first row of each sequence
    int* len = st + B + 1;           // [B] tokens it holds
    int* base = len + B;             // [B] first tile of each sequence among its kind's; the kind in bit 31
    const int pl = a.prefix_len ? min(max(__ldg(a.prefix_len), 0), d.pre_pages * d.ps) : 0;
    const int cap = pl + d.own_pages * d.ps;
    // starts: running maximum of the given ones, within [0, T]
    {
        int run = 0;
        for (int i0 = 0; i0 <= B; i0 += kPlanThreads) {
            const int i = i0 + tid;
            const int v = i <= B ? min(max(__ldg(a.q_start + i), 0), d.T) : 0;
            int all;
            const int exc = block_scan(v, 0, ibuf, &all, [](int x, int y) { return max(x, y); });
            if (i <= B) st[i] = max(run, max(exc, v));
            run = max(run, all);
        }
        for (int i = tid; i < B; i += kPlanThreads) len[i] = min(max(__ldg(a.kv_len + i), 0), cap);
    }
    __syncthreads();
    // position of row t of sequence b; -1 for all before its first (a window's start behind that stays within 32 bits)
    auto pos_of = [&](int b, int t) { return max(-1, len[b] - st[b + 1] + t); };
    const int r_lo = st[0] * G, r_hi = st[B] * G;
    const bool pre_many = r_hi - r_lo > d.few;
    const int pre_rows = pre_many ? kRowsP : kRowsS;
    const int pre_tiles = pl > 0 ? (r_hi - r_lo + pre_rows - 1) / pre_rows : 0;
    auto alone = [&](int b) { return (st[b + 1] - st[b]) * G > kRowsAlone; };
    auto many_of = [&](int b) { return (st[b + 1] - st[b]) * G > d.few; };
    // first tile of each sequence: the prefix's come first
    int nt[2] = {pre_many ? 0 : pre_tiles, pre_many ? pre_tiles : 0};
    for (int i0 = 0; i0 < B; i0 += kPlanThreads) {
        const int b = i0 + tid;
        const int rows = b < B ? (st[b + 1] - st[b]) * G : 0;
        const bool many = b < B && many_of(b);
        int all0, all1;
        const auto add = [](int x, int y) { return x + y; };
        const int e0 = block_scan(many ? 0 : (rows + kRowsS - 1) / kRowsS, 0, ibuf, &all0, add);
        const int e1 = block_scan(many ? (rows + kRowsP - 1) / kRowsP : 0, 0, ibuf, &all1, add);
        if (b < B) base[b] = many ? (int)(0x80000000u | (unsigned)(nt[1] + e1)) : nt[0] + e0;
        nt[0] += all0;
        nt[1] += all1;
    }
    __syncthreads();

    // ---- per token and per row
    const int gtid = blockIdx.x * kPlanThreads + tid, gn = gridDim.x * kPlanThreads;
    for (int t = gtid; t < d.T; t += gn) {
        const bool live = t >= st[0] && t < st[B];
        int b = -1, pos = -1;
        if (live) {
            b = seq_of(st, B, t);
            pos = pos_of(b, t);
        }
        at<int>(a.plan, d.tok_seq)[t] = b;
        at<int>(a.plan, d.tok_pos)[t] = pos;
    }
    for (int r = gtid; r < d.T * G; r += gn) {
        int pre = -1;                // the row's prefix tile: kind in bit 31
        if (pre_tiles && r >= r_lo && r < r_hi && !alone(seq_of(st, B, r / G)))
            pre = (int)((pre_many ? 0x80000000u : 0u) | (unsigned)((r - r_lo) / pre_rows));
        at<int>(a.plan, d.row_pre)[r] = pre;
    }
    if (blockIdx.x != 0) return;

    // ---- the tiles, by CTA 0
    auto first_key = [&](int pos) { return d.window > 0 ? max(0, pos + 1 - d.window) : 0; };
    for (int i = tid; i < pre_tiles; i += kPlanThreads) {
        Tile t{};
        t.row0 = r_lo + i * pre_rows;
        t.nrows = min(pre_rows, r_hi - t.row0);
        t.seq = -1;
        // the positions of the rows that have no tile of both segments: within a sequence they rise
        const int t0 = t.row0 / G, t1 = (t.row0 + t.nrows - 1) / G;
        int lo = 0x7fffffff, hi = 0;
        for (int b = seq_of(st, B, t0); b < B && st[b] <= t1; b++) {
            const int f = max(t0, st[b]), l = min(t1, st[b + 1] - 1);
            if (l < f || alone(b)) continue;
            lo = min(lo, first_key(pos_of(b, f)));
            hi = max(hi, pos_of(b, l) + 1);
        }
        t.lo1 = lo / kUnit * kUnit;
        t.hi1 = min(pl, hi);
        t.n = t.n1 = max(0, (t.hi1 - t.lo1 + kUnit - 1) / kUnit);
        at<Tile>(a.plan, d.tiles[pre_many ? 1 : 0])[i] = t;
    }
    // each sequence names its tiles (a warp per sequence: a long prompt has many)
    for (int b = tid >> 5; b < B; b += kPlanThreads / 32) {
        const bool many = many_of(b);
        const int br = many ? kRowsP : kRowsS, n = ((st[b + 1] - st[b]) * G + br - 1) / br;
        Tile* tiles = at<Tile>(a.plan, d.tiles[many ? 1 : 0]) + ((unsigned)base[b] & 0x7fffffffu);
        for (int k = tid & 31; k < n; k += 32) tiles[k].seq = b;
    }
    __syncthreads();
    Hdr* h = reinterpret_cast<Hdr*>(a.plan);
    for (int kind = 0; kind < 2; kind++) {
        Tile* tiles = at<Tile>(a.plan, d.tiles[kind]);
        const int br = kind ? kRowsP : kRowsS;
        const bool pre_here = pre_tiles > 0 && (kind == 1) == pre_many;
        const auto add = [](long long x, long long y) { return x + y; };
        const int heads = d.nkv * (kind ? d.cs : 1), ctas = d.ctas[kind];
        long long work = 0, filled = 0;      // units of one head, tiles that have any
        for (int i0 = 0; i0 < nt[kind]; i0 += kPlanThreads) {
            const int i = i0 + tid;
            Tile t{};
            if (i < nt[kind]) {
                if (pre_here && i < pre_tiles) {
                    t = tiles[i];
                } else {
                    const int b0 = tiles[i].seq;
                    const int lr = (i - (int)((unsigned)base[b0] & 0x7fffffffu)) * br;
                    t.seq = b0;
                    t.row0 = st[b0] * G + lr;
                    t.nrows = min(br, (st[b0 + 1] - st[b0]) * G - lr);
                    const int p0 = pos_of(b0, t.row0 / G), p1 = pos_of(b0, (t.row0 + t.nrows - 1) / G);
                    t.lo2 = max(0, first_key(p0) - pl) / kUnit * kUnit;
                    t.hi2 = p1 + 1 - pl;
                    t.n = max(0, (t.hi2 - t.lo2 + kUnit - 1) / kUnit);
                    if (kind == 1 && alone(b0)) {
                        t.lo1 = first_key(p0) / kUnit * kUnit;
                        t.hi1 = min(pl, p1 + 1);
                        t.n1 = max(0, (t.hi1 - t.lo1 + kUnit - 1) / kUnit);
                        t.n += t.n1;
                    }
                    t.solo = 1;
                    if (pre_tiles && !(kind && alone(b0))) {
                        const Tile* pt = at<Tile>(a.plan, d.tiles[pre_many ? 1 : 0]);
                        for (int j = (t.row0 - r_lo) / pre_rows; j <= (t.row0 + t.nrows - 1 - r_lo) / pre_rows; j++)
                            if (pt[j].n > 0) t.solo = 0;
                    }
                }
            }
            if (i < nt[kind]) tiles[i] = t;
            long long all;
            block_scan((long long)t.n, 0LL, wbuf, &all, add);
            work += all;
            block_scan(t.n > 0 ? 1LL : 0LL, 0LL, wbuf, &all, add);
            filled += all;
        }
        __syncthreads();
        // Equal stretches of the line of all heads' units, wherever their borders fall; or, if every tile can have
        // CTAs of its own, the shortest stretch for which they suffice when each tile starts at a border.
        const int cost = kind ? kTileCostP : kTileCostS;
        long long u = max(1LL, (work * heads + ctas - 1) / ctas);
        bool aligned = false;
        {
            auto stretches = [&](long long len) {
                long long n = 0;
                for (int i = tid; i < nt[kind]; i += kPlanThreads) n += (tiles[i].n + len - 1) / len;
                long long all;
                block_scan(n, 0LL, wbuf, &all, add);
                return all * heads;
            };
            const long long most = u + (kind ? kBorderCostP : kBorderCostS);
            if (work > 0 && stretches(most) <= ctas) {
                long long lo = u, hi = most;
                while (lo < hi) {
                    const long long m = (lo + hi) / 2;
                    if (stretches(m) <= ctas) hi = m;
                    else lo = m + 1;
                }
                u = lo;
                aligned = true;
            } else {
                u = max(1LL, ((work + (long long)cost * filled) * heads + ctas - 1) / ctas);
            }
        }
        long long run = 0;
        for (int i0 = 0; i0 < nt[kind]; i0 += kPlanThreads) {
            const int i = i0 + tid;
            const int n = i < nt[kind] ? tiles[i].n : 0;
            const int idle = aligned ? (int)((u - n % u) % u) : n > 0 ? cost : 0;
            long long all;
            const long long exc = block_scan((long long)n + idle, 0LL, wbuf, &all, add);
            if (i < nt[kind]) {
                tiles[i].off = run + exc;
                tiles[i].idle = idle;
            }
            run += all;
        }
        __syncthreads();
        const long long total = run * heads;
        if (tid == 0) {
            h->nt[kind] = nt[kind];
            h->wt[kind] = run;
            h->u[kind] = u;
        }
        // What is left to the join kernel: groups of 1, 2, 4 or 8 rows, the smallest of which there is one per CTA at
        // most (a CTA's warps share a group's rows), or 8.
        if (tid == 0) s_joins = 0;
        if (tid < 4) s_rows[tid] = 0;
        __syncthreads();
        auto left_of = [&](int i) {          // rows left of tile i / nkv for KV head i % nkv
            const Tile& t = tiles[i / d.nkv];
            if (t.seq < 0) return 0;
            const int walks = kind ? d.cs : 1, head = i % d.nkv;
            bool left = !(t.solo && t.n > 0);
            for (int k = 0; k < walks && !left; k++) {
                const Span sp = span_of((long long)(head * walks + k) * run + t.off, t.n, u);
                left = sp.c0 != sp.c1;
            }
            return left ? t.nrows : 0;
        };
        const int pairs = nt[kind] * d.nkv;
        for (int i = tid; i < pairs; i += kPlanThreads) {
            const int n = left_of(i);
            for (int k = 0; k < 4 && n > 0; k++) atomicAdd(&s_rows[k], (n + (1 << k) - 1) >> k);
        }
        __syncthreads();
        int lr = 0;
        while (lr < 3 && s_rows[lr] > d.join_ctas) lr++;
        for (int i = tid; i < pairs; i += kPlanThreads) {
            const int n = (left_of(i) + (1 << lr) - 1) >> lr;
            const int at0 = n > 0 ? atomicAdd(&s_joins, n) : 0;
            for (int k = 0; k < n; k++) at<int2>(a.plan, d.joins[kind])[at0 + k] = make_int2(i / d.nkv, k << 16 | i % d.nkv);
        }
        __syncthreads();
        if (tid == 0) {
            h->nj[kind] = s_joins;
            h->rj[kind] = 1 << lr;
        }
        for (int c = tid; c < d.ctas[kind]; c += kPlanThreads) {
            Start s{};
            s.head = -1;
            const long long at0 = (long long)c * u;
            if (at0 < total) {
                const long long rem = at0 % run;
                s.head = (int)(at0 / run);
                int lo = 0, hi = nt[kind];       // the last tile with off <= rem; of equal ones it is the one with units
                while (hi - lo > 1) {
                    const int m = (lo + hi) >> 1;
                    if (tiles[m].off <= rem) lo = m;
                    else hi = m;
                }
                s.tile = lo;
                s.unit = (int)(rem - tiles[lo].off);
                if (s.unit >= tiles[lo].n) {     // between two tiles
                    s.skip = tiles[lo].n + tiles[lo].idle - s.unit;
                    s.unit = 0;
                    if (++s.tile == nt[kind]) {
                        s.tile = 0;
                        s.head++;
                    }
                    if (s.skip >= u || at0 + s.skip >= total) s.head = -1;
                }
                s.t = tiles[s.tile];
            }
            at<Start>(a.plan, d.start[kind])[c] = s;
        }
    }
    if (tid == 0) {
        h->key = d.key;
        h->prefix_len = pl;
        h->tok_lo = st[0];
        h->tok_hi = st[B];
    }
}

// ------------------------------------------------------------------ append
struct AppendArgs {
    const void* plan;
    const void* qkv;
    const float* qnw;
    const float* knw;
    const float* cos_t;
    const float* sin_t;
    uint16_t* kc;
    uint16_t* vc;
    const int* table;
    uint16_t* q_out;
    long long row_stride, q_stride;
    int koff, voff, num_pages;
    Dims d;
};

constexpr int kAppendThreads = 256;

template <int N, bool F32>
__device__ __forceinline__ void load_n(const void* base, long long e, float (&v)[N]) {
    if constexpr (F32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + e);
        #pragma unroll
        for (int j = 0; j < N / 4; j++) {
            const float4 x = __ldg(p + j);
            v[4 * j] = x.x; v[4 * j + 1] = x.y; v[4 * j + 2] = x.z; v[4 * j + 3] = x.w;
        }
    } else {
        const __half* p = reinterpret_cast<const __half*>(base) + e;
        #pragma unroll
        for (int j = 0; j < N; j += 8) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if constexpr (N >= 8) u = __ldg(reinterpret_cast<const uint4*>(p + j));
            else *reinterpret_cast<uint2*>(&u) = __ldg(reinterpret_cast<const uint2*>(p));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            #pragma unroll
            for (int i = 0; i < (N < 8 ? N : 8); i++) v[j + i] = i & 1 ? h_hi(w[i / 2]) : h_lo(w[i / 2]);
        }
    }
}

template <int N>
__device__ __forceinline__ void store_half(uint16_t* p, const float (&v)[N]) {
    uint32_t w[N / 2];
    #pragma unroll
    for (int j = 0; j < N / 2; j++) w[j] = half_pair(v[2 * j], v[2 * j + 1]);
    if constexpr (N == 4) {
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
        #pragma unroll
        for (int j = 0; j < N / 8; j++)
            reinterpret_cast<uint4*>(p)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    }
}

// Few tokens, or few heads: one warp per head, a token's heads over several CTAs (blockIdx.y); latency is what counts.
// Lane l holds elements l * PER .. of the head; element i's rotation partner i +- hd/2 is in lane l ^ 16.
template <int HD, bool XF32>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
    constexpr int PER = HD / 32;
    const Dims& d = a.d;
    const Hdr* h = hdr_of(a.plan);
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    const int j = blockIdx.y * (kAppendThreads / 32) + (threadIdx.x >> 5);
    const bool is_q = j < d.nH, is_v = j >= d.nH + d.nkv;
    const int kv = is_v ? j - d.nH - d.nkv : j - d.nH;
    if (j >= d.nH + 2 * d.nkv) return;
    // the head, before it is known where it goes: that is a chain of three loads
    float v[PER];
    load_n<PER, XF32>(a.qkv, (long long)t * a.row_stride + lane * PER +
                      (is_q ? (long long)j * HD : (is_v ? a.voff : a.koff) + (long long)kv * HD), v);
    const bool fits = plan_fits(h, d);
    const int prefix_len = h->prefix_len;
    const int b = __ldg(at<int>(a.plan, d.tok_seq) + t), pos = __ldg(at<int>(a.plan, d.tok_pos) + t);
    if (!fits) {
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(&g_status_paged, kStatusPlan);
        return;
    }
    if (b < 0 || pos < 0) return;    // behind the last sequence; or more new tokens than its length says
    int slot = -1;                   // the token's row of the cache for KV head 0
    if (pos >= prefix_len) {
        const int own = pos - prefix_len;
        slot = cache_row(__ldg(a.table + (size_t)b * d.own_pages + (own >> d.lps)), a.num_pages, d.nkv, d.lps, 0, own);
    }
    if (!is_q && slot < 0) return;
    float ss = 0.f;
    #pragma unroll
    for (int i = 0; i < PER; i++) ss = fmaf(v[i], v[i], ss);
    #pragma unroll
    for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    const float r = rsqrtf(ss / (float)HD + kEps);
    if (is_v) {
        #pragma unroll
        for (int i = 0; i < PER; i++) v[i] *= r;
    } else {
        float cs[PER], sn[PER], g[PER];
        load_n<PER, true>(a.cos_t, (long long)pos * HD + lane * PER, cs);
        load_n<PER, true>(a.sin_t, (long long)pos * HD + lane * PER, sn);
        load_n<PER, true>(is_q ? a.qnw : a.knw, lane * PER, g);
        #pragma unroll
        for (int i = 0; i < PER; i++) {
            const float n = v[i] * r * g[i];
            const float o = __shfl_xor_sync(0xffffffffu, n, 16);
            v[i] = n * cs[i] + (lane < 16 ? -o : o) * sn[i];
        }
    }
    uint16_t* dst = is_q ? a.q_out + (long long)t * a.q_stride + (long long)j * HD
                         : (is_v ? a.vc : a.kc) + ((long long)slot + kv * d.ps) * HD;
    store_half<PER>(dst + lane * PER, v);
}

// Many tokens of many heads: HBM-bound on q|k|v in and out, so the rows stream through shared memory.  A warp of each persistent
// CTA copies a token's q, k, v and rotation rows into a ring of stages (bulk copies, 32 tokens' places looked up
// at once), the others take the heads from there.  Lane l holds elements l * PER/2 .. of both halves of a head, so that
// both ends of a rotation are its own.  Five prompts of 300 to 1,600 tokens, 129 MB in and out: 32 us, 0.61 of the measured
// copy rate; what is left is the head warps' own work (the sums across lanes, two heads a token one after the other) with
// 56 registers each, and the first rows' way through the plan and the table.
// head warps of a CTA, by what their registers leave room for twice per SM
constexpr int stream_warps(int hd) { return hd == 512 ? 8 : 16; }
constexpr int kStreamSmem = 110 * 1024;     // its ring: two CTAs' fit an SM

template <int N, bool F32>
__device__ __forceinline__ void lds_n(uint32_t at, float* v) {   // N = 2, 4, 8 elements
    if constexpr (F32) {
        #pragma unroll
        for (int j = 0; j < N; j += 4) {
            if constexpr (N >= 4)
                asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v[j]), "=f"(v[j + 1]), "=f"(v[j + 2]),
                             "=f"(v[j + 3]) : "r"(at + 4 * j) : "memory");
            else
                asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(at) : "memory");
        }
    } else {
        uint32_t w[N / 2];
        if constexpr (N == 8)
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
        else if constexpr (N == 4)
            asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
        else
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
        #pragma unroll
        for (int i = 0; i < N; i++) v[i] = i & 1 ? h_hi(w[i / 2]) : h_lo(w[i / 2]);
    }
}
template <int N>
__device__ __forceinline__ void store_half_n(uint16_t* p, const float* v) {
    uint32_t w[N / 2];
    #pragma unroll
    for (int j = 0; j < N / 2; j++) w[j] = half_pair(v[2 * j], v[2 * j + 1]);
    if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (N == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
}

// bytes of a stage: the heads, then the two rotation rows
__host__ __device__ inline int stage_bytes(const Dims& d, int esz) { return (d.nH + 2 * d.nkv) * d.hd * esz + 2 * d.hd * 4; }

template <int HD, bool XF32>
__global__ void __launch_bounds__(32 * (stream_warps(HD) + 1), HD == 512 ? 1 : 2) append_stream_kernel(const AppendArgs a, int stages) {
    constexpr int kStreamWarps = stream_warps(HD);
    constexpr int PER = HD / 32, HP = PER / 2, ESZ = XF32 ? 4 : 2;
    extern __shared__ __align__(128) uint8_t ring_raw[];
    __shared__ __align__(8) uint64_t bars[2 * 8];
    __shared__ int s_slot[8], s_abort;
    const Dims& d = a.d;
    const Hdr* h = hdr_of(a.plan);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (!plan_fits(h, d)) {
        if (blockIdx.x == 0 && tid == 0) atomicOr(&g_status_paged, kStatusPlan);
        return;
    }
    const uint32_t ring = smem_u32(ring_raw), bar0 = smem_u32(bars);
    const int bytes = stage_bytes(d, ESZ);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (8 + s); };
    if (tid == 0) {
        for (int s = 0; s < 8; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), kStreamWarps);
        }
        fence_mbar_init();
        s_abort = 0;
    }
    __syncthreads();
    volatile int* abort = &s_abort;
    const int lo = h->tok_lo, hi = h->tok_hi, prefix_len = h->prefix_len;   // the rows that belong to a sequence
    const int first = lo + blockIdx.x, step = gridDim.x;
    const int nq = d.nH * HD, nk = d.nkv * HD;
    if (warp == kStreamWarps) {
        int slot = -1, pos = -1, s = 0, used = 0;
        uint32_t turn = 0;
        bool ok = true;
        for (int t = first, n = 0; t < hi; t += step, n++) {
            if ((n & 31) == 0) {     // the places of this CTA's next 32 tokens
                const long long mine = t + (long long)lane * step;
                pos = slot = -1;
                if (mine < hi) {
                    const int b = __ldg(at<int>(a.plan, d.tok_seq) + mine);
                    pos = __ldg(at<int>(a.plan, d.tok_pos) + mine);
                    const int own = pos - prefix_len;
                    if (b >= 0 && pos >= 0 && own >= 0)
                        slot = cache_row(__ldg(a.table + (size_t)b * d.own_pages + (own >> d.lps)), a.num_pages, d.nkv, d.lps, 0, own);
                }
            }
            const int p = __shfl_sync(0xffffffffu, pos, n & 31), c = __shfl_sync(0xffffffffu, slot, n & 31);
            if (used == stages) ok = __all_sync(0xffffffffu, wait_short(empty(s), turn ^ 1u, abort, &g_status_paged));
            if (!ok) break;
            if (lane == 0) {
                s_slot[s] = p < 0 ? -2 : c;            // -2: no position, nothing to do; -1: its q only
                const uint32_t dst = ring + s * bytes;
                const char* src = reinterpret_cast<const char*>(a.qkv) + (long long)t * a.row_stride * ESZ;
                // every stage is filled whole, so its count is always the same
                const long long rot = (long long)max(p, 0) * HD;
                mbar_arrive_expect_tx(full(s), bytes);
                bulk_g2s_nohint(dst, src, nq * ESZ, full(s));
                bulk_g2s_nohint(dst + nq * ESZ, src + (long long)a.koff * ESZ, nk * ESZ, full(s));
                bulk_g2s_nohint(dst + (nq + nk) * ESZ, src + (long long)a.voff * ESZ, nk * ESZ, full(s));
                bulk_g2s_nohint(dst + (nq + 2 * nk) * ESZ, a.cos_t + rot, HD * 4, full(s));
                bulk_g2s_nohint(dst + (nq + 2 * nk) * ESZ + HD * 4, a.sin_t + rot, HD * 4, full(s));
            }
            __syncwarp();
            used = max(used, s + 1);
            if (++s == stages) {
                s = 0;
                turn ^= 1u;
            }
        }
        // what is in flight lands before the CTA gives up its shared memory, whoever gives up waiting for it
        for (int k = 0; k < used; k++) mbar_wait_drain(full(k), k < s ? turn : turn ^ 1u, &g_status_paged);
        return;
    }
    const int heads = d.nH + 2 * d.nkv;
    float gq[PER], gk[PER];          // the norm weights of this lane's elements
    #pragma unroll
    for (int e = 0; e < 2; e++)
        #pragma unroll
        for (int i = 0; i < HP; i++) {
            gq[e * HP + i] = __ldg(a.qnw + e * (HD / 2) + lane * HP + i);
            gk[e * HP + i] = __ldg(a.knw + e * (HD / 2) + lane * HP + i);
        }
    int s = 0;
    uint32_t turn = 0;
    for (int t = first; t < hi; t += step) {
        if (!__all_sync(0xffffffffu, wait_short(full(s), turn, abort, &g_status_paged))) break;
        const int slot = *(volatile int*)&s_slot[s];
        const uint32_t base = ring + s * bytes, rot = base + (nq + 2 * nk) * ESZ;
        float cs[PER], sn[PER];
        #pragma unroll
        for (int e = 0; e < 2; e++) {
            lds_n<HP, true>(rot + (e * (HD / 2) + lane * HP) * 4, cs + e * HP);
            lds_n<HP, true>(rot + HD * 4 + (e * (HD / 2) + lane * HP) * 4, sn + e * HP);
        }
        for (int j = warp; j < heads && slot > -2; j += kStreamWarps) {
            const bool is_q = j < d.nH, is_v = j >= d.nH + d.nkv;
            const int kv = is_v ? j - d.nH - d.nkv : j - d.nH;
            if (!is_q && slot < 0) break;
            float v[PER], ss = 0.f;
            #pragma unroll
            for (int e = 0; e < 2; e++) lds_n<HP, XF32>(base + (j * HD + e * (HD / 2) + lane * HP) * ESZ, v + e * HP);
            #pragma unroll
            for (int i = 0; i < PER; i++) ss = fmaf(v[i], v[i], ss);
            #pragma unroll
            for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            const float r = rsqrtf(ss / (float)HD + kEps);
            #pragma unroll
            for (int i = 0; i < PER; i++) v[i] *= is_v ? r : r * (is_q ? gq[i] : gk[i]);
            if (!is_v) {
                #pragma unroll
                for (int i = 0; i < HP; i++) {
                    const float x = v[i], y = v[HP + i];
                    v[i] = x * cs[i] - y * sn[i];
                    v[HP + i] = y * cs[HP + i] + x * sn[HP + i];
                }
            }
            uint16_t* dst = is_q ? a.q_out + (long long)t * a.q_stride + (long long)j * HD
                                 : (is_v ? a.vc : a.kc) + ((long long)slot + kv * d.ps) * HD;
            #pragma unroll
            for (int e = 0; e < 2; e++) store_half_n<HP>(dst + e * (HD / 2) + lane * HP, v + e * HP);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
        if (++s == stages) {
            s = 0;
            turn ^= 1u;
        }
    }
}

// ------------------------------------------------------------------ attention, few rows
// A tile of up to 8 rows (the query heads of a token or two) over a stretch of keys, HBM-bound on them.  The
// products are transposed so that the rows are the n = 8 of m16n8k16 and the keys or the head's elements
// the m = 16:
//   S^T [16 keys x 8 rows] = K [16 x hd] Q^T,   O^T [hd x 8] += V^T [hd x 16 keys] P^T
// K and V fragments come from shared memory by ldmatrix (transposed for V), Q stays in registers, and P^T
// gets from its accumulator layout to an operand's by movmatrix.  P enters as f16 hi + lo, since these
// MMAs are not what bounds the kernel, and 2^15 times too large, as far as f16 goes: a weight then counts down to 2^-40 of
// the row's largest (without that to 2^-25: a hundred thousand keys just below are lost, a percent of a long row).  The
// four warps of a CTA take every fourth block of 16 keys, each with its own ring of TMA-filled buffers, its own running maximum and sum: no CTA barrier until the
// partials of the warps are added at a piece's end.  48 decode tokens over 868 MB of ragged keys and values: 140 us, 0.95
// of the measured copy rate.
constexpr int kFewWarps = 4;
constexpr float kFewLift = 15.f, kFewDrop = 0x1p-15f;
constexpr int kBlk = 16;             // keys per block (one page always holds a block: page_size >= 16)

template <int HD>
struct FewCfg {
    static constexpr int ENTRY = kBlk * HD * 2;               // bytes of a block of K or of V
    static constexpr int NST = HD == 128 ? 6 : 3;             // ring entries per warp: 24 / 24 / 48 KB
    static constexpr int SMEM = kFewWarps * NST * ENTRY + 1024;   // + alignment
    static constexpr int PITCH = HD + 4;                      // floats per row of the merge buffer
    static_assert(kRowsS * PITCH * 4 <= NST * ENTRY, "a warp's partial fits its ring");
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movm_t(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int HD>
__global__ void __launch_bounds__(32 * kFewWarps, HD == 512 ? 1 : 2)
few_kernel(const Args a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using C = FewCfg<HD>;
    constexpr int KK = HD / 16;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[kFewWarps][C::NST];
    __shared__ float s_m[kFewWarps][kRowsS], s_l[kFewWarps][kRowsS];
    __shared__ int s_abort;
    const Dims& d = a.d;
    const Hdr* h = hdr_of(a.plan);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
    pdl_launch_dependents();
    if (!plan_fits(h, d)) {
        if (blockIdx.x == 0 && tid == 0) atomicOr(&g_status_paged, kStatusPlan);
        pdl_wait();
        return;
    }
    const Start& st = at<Start>(a.plan, d.start[0])[blockIdx.x];
    Tile t = st.t;
    bool first = true;
    if (st.head < 0) {
        pdl_wait();
        return;
    }
    const uint32_t ring = ((smem_u32(smem_raw) + 1023u) & ~1023u) + (uint32_t)(warp * C::NST * C::ENTRY);
    uint8_t* ring_p = smem_raw + (ring - smem_u32(smem_raw));
    const uint32_t bar0 = smem_u32(&bars[warp][0]);
    if (lane == 0) {
        for (int i = 0; i < C::NST; i++) mbar_init(bar0 + 8 * i, 1);
        fence_mbar_init();
    }
    if (tid == 0) s_abort = 0;
    __syncthreads();
    volatile int* abort = &s_abort;
    const int pl = h->prefix_len, G = d.G;
    const long long wt = h->wt[0], u_all = h->u[0];
    const int ntiles = h->nt[0];
    const Tile* tiles = at<Tile>(a.plan, d.tiles[0]);
    const int* tok_pos = at<int>(a.plan, d.tok_pos);
    long long left = min(u_all, wt * d.nkv - (long long)blockIdx.x * u_all) - st.skip;
    int head = st.head, ti = st.tile, unit = st.unit;
    int entry = 0;                       // ring position of the next entry to consume; runs on over pieces
    uint32_t phase = 0;                  // parity bit per ring position

    while (left > 0) {
        if (ti == ntiles) {
            ti = 0;
            head++;
        }
        if (!first) t = tiles[ti];
        first = false;
        if (t.n == 0) {
            ti++;
            unit = 0;
            continue;
        }
        const int nu = (int)min((long long)(t.n - unit), left);
        const Unit un0 = unit_of(t, unit);                           // a few-rows tile has one segment
        const int key0 = un0.key, key1 = min(un0.hi, key0 + nu * kUnit);
        const int kbase = t.seq < 0 ? 0 : pl;                        // position of the segment's key 0
        const int* table = t.seq < 0 ? a.pre_table : a.table + (size_t)t.seq * d.own_pages;
        const int table_n = t.seq < 0 ? d.pre_pages : d.own_pages;
        // this thread's rows: 2 * q4 and 2 * q4 + 1 of the scores; row g of Q
        int vlo[2], vhi[2], all_lo = 0, all_hi = 0x7fffffff;         // keys that a row sees; that all rows see
        #pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = 2 * q4 + i;
            const int pos = __ldg(tok_pos + (t.row0 + min(r, t.nrows - 1)) / G);
            vhi[i] = pos + 1 - kbase;
            vlo[i] = d.window > 0 ? pos + 1 - d.window - kbase : 0;
            all_lo = max(all_lo, vlo[i]);
            all_hi = min(all_hi, vhi[i]);
        }
        #pragma unroll
        for (int m = 1; m <= 2; m <<= 1) {
            all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, m));
            all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, m));
        }
        const int tok_a = t.row0 / G, tok_b = (t.row0 + t.nrows - 1) / G;
        uint32_t qf[KK][2];
        {
            const bool live = g < t.nrows;
            const int row = t.row0 + (live ? g : 0);
            const uint16_t* qp = a.q + (long long)(row / G) * a.q_stride + (long long)(head * G + row % G) * HD + 2 * q4;
            #pragma unroll
            for (int k = 0; k < KK; k++) {
                qf[k][0] = live ? __ldg(reinterpret_cast<const uint32_t*>(qp + 16 * k)) : 0u;
                qf[k][1] = live ? __ldg(reinterpret_cast<const uint32_t*>(qp + 16 * k + 8)) : 0u;
            }
        }
        float o[KK][4];
        #pragma unroll
        for (int k = 0; k < KK; k++) o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        // this warp's blocks: key0 + 16 * (warp + 4 n)
        const int nblk_all = (key1 - key0 + kBlk - 1) / kBlk;
        const int nblk = (nblk_all - warp + kFewWarps - 1) / kFewWarps;
        const int total = 2 * max(nblk, 0);      // entries: K and V of each block in turn
        uint32_t valid = 0;                      // bit n % 32: block n's page exists
        int ids = 0, ids_at = -32;               // page ids of 32 blocks, one per lane
        int eslot = entry, issued = 0;
        auto issue = [&](int e) {                // whole warp; e counts the piece's entries
            const int n = e >> 1;
            if (n >= ids_at + 32) {
                ids_at = n;
                const int key = key0 + kBlk * (warp + kFewWarps * (n + lane));
                const int page = key >> d.lps;
                ids = key < key1 && page < table_n ? __ldg(table + page) : -1;
            }
            const int key = key0 + kBlk * (warp + kFewWarps * n);
            const int page = __shfl_sync(0xffffffffu, ids, n - ids_at);
            const int at_row = cache_row(page, a.num_pages, d.nkv, d.lps, head, key);
            const bool ok = at_row >= 0;
            if (!(e & 1)) valid = (valid & ~(1u << (n & 31))) | ((ok ? 1u : 0u) << (n & 31));
            // a page that is not there: past the map's last row, which TMA fills with zeros
            const int row = ok ? at_row : a.num_pages * d.nkv * d.ps;
            if (lane == 0) {
                const uint32_t bar = bar0 + 8 * eslot;
                mbar_arrive_expect_tx(bar, C::ENTRY);
                tma_chunks(ring + (uint32_t)(eslot * C::ENTRY), (e & 1) ? &vmap : &kmap, row, 0, bar);
            }
            eslot = eslot + 1 == C::NST ? 0 : eslot + 1;
            issued++;
        };
        const int ahead = min(C::NST, total);
        for (int e = 0; e < ahead; e++) issue(e);
        bool ok = true;
        int done = 0;                            // entries consumed
        auto next = [&]() {                      // wait for the next entry; its address
            ok = __all_sync(0xffffffffu, wait_short(bar0 + 8 * entry, (phase >> entry) & 1u, abort, &g_status_paged));
            if (ok) phase ^= 1u << entry;
            return ring + (uint32_t)(entry * C::ENTRY);
        };
        auto release = [&]() {                   // the entry just read may be filled again
            __syncwarp();
            entry = entry + 1 == C::NST ? 0 : entry + 1;
            done++;
            if (done + C::NST - 1 < total) issue(done + C::NST - 1);
        };
        for (int n = 0; n < nblk; n++) {
            const int key = key0 + kBlk * (warp + kFewWarps * n);
            const uint32_t kb = next();
            if (!ok) break;
            float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};   // two chains
            {
                const int row = (lane & 7) + 8 * ((lane >> 3) & 1);
                #pragma unroll
                for (int k = 0; k < KK; k++) {
                    uint32_t f[4];
                    const int un = 2 * k + (lane >> 4);
                    ldsm4(kb + (un >> 3) * (kBlk * 128) + row * 128 + (((un & 7) ^ (row & 7)) << 4), f);
                    mma8(s[k & 1], f, qf[k][0], qf[k][1]);
                }
            }
            const bool there = (valid >> (n & 31)) & 1u;
            release();
            // keys g and g + 8 of rows 2 q4 and 2 q4 + 1
            float x[4];
            #pragma unroll
            for (int e = 0; e < 4; e++) x[e] = (s[0][e] + s[1][e]) * a.scale;
            const bool edge = !there || key < all_lo || key + kBlk > min(all_hi, key1);
            if (edge) {
                #pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = key + g + 8 * (e >> 1);
                    if (!there || j >= key1 || j < vlo[e & 1] || j >= vhi[e & 1]) x[e] = -INFINITY;
                }
            }
            float corr[2];
            #pragma unroll
            for (int i = 0; i < 2; i++) {
                float mx = fmaxf(x[i], x[2 + i]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float mn = fmaxf(m[i], mx);
                const float mu = mn == -INFINITY ? 0.f : mn;     // nothing seen yet: weights 2^-inf = 0
                corr[i] = exp2_approx(m[i] - mu);
                m[i] = mn;
                // (the difference first: at scores far from zero a base less 15 may be no f32)
                x[i] = exp2_approx(x[i] - mu + kFewLift);
                x[2 + i] = exp2_approx(x[2 + i] - mu + kFewLift);
                l[i] = fmaf(l[i], corr[i], x[i] + x[2 + i]);
            }
            const __half2 h0 = __floats2half2_rn(x[0], x[1]), h1 = __floats2half2_rn(x[2], x[3]);
            const __half2 r0 = __floats2half2_rn(x[0] - __low2float(h0), x[1] - __high2float(h0));
            const __half2 r1 = __floats2half2_rn(x[2] - __low2float(h1), x[3] - __high2float(h1));
            const uint32_t ph0 = movm_t(*reinterpret_cast<const uint32_t*>(&h0));
            const uint32_t ph1 = movm_t(*reinterpret_cast<const uint32_t*>(&h1));
            const uint32_t pw0 = movm_t(*reinterpret_cast<const uint32_t*>(&r0));
            const uint32_t pw1 = movm_t(*reinterpret_cast<const uint32_t*>(&r1));
            if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
                #pragma unroll
                for (int k = 0; k < KK; k++) {
                    o[k][0] *= corr[0];
                    o[k][1] *= corr[1];
                    o[k][2] *= corr[0];
                    o[k][3] *= corr[1];
                }
            }
            const uint32_t vb = next();
            if (!ok) break;
            const int row = (lane & 7) + 8 * (lane >> 4);
            auto vfrag = [&](int k, uint32_t (&f)[4]) {
                const int un = 2 * k + ((lane >> 3) & 1);
                ldsm4t(vb + (un >> 3) * (kBlk * 128) + row * 128 + (((un & 7) ^ (row & 7)) << 4), f);
            };
            if (!edge) {
                #pragma unroll
                for (int k = 0; k < KK; k++) {
                    uint32_t f[4];
                    vfrag(k, f);
                    mma8(o[k], f, ph0, ph1);
                    mma8(o[k], f, pw0, pw1);
                }
            } else {
                // A value behind the mask may be anything, NaN included, and 0 x NaN is not 0: the values a
                // token does not see are cleared.  Rows of several tokens see different keys, so each token
                // then has products of its own, of which only its rows are added.
                for (int tok = tok_a; tok <= tok_b; tok++) {
                    const int pos = __ldg(tok_pos + tok);
                    const int th = min(key1, pos + 1 - kbase), tl = d.window > 0 ? pos + 1 - d.window - kbase : 0;
                    auto keep = [&](int j) { return there && j >= tl && j < th; };
                    const int j0 = key + 2 * q4;
                    const uint32_t k0 = (keep(j0) ? 0xffffu : 0u) | (keep(j0 + 1) ? 0xffff0000u : 0u);
                    const uint32_t k1 = (keep(j0 + 8) ? 0xffffu : 0u) | (keep(j0 + 9) ? 0xffff0000u : 0u);
                    const bool c0 = (t.row0 + 2 * q4) / G == tok, c1 = (t.row0 + 2 * q4 + 1) / G == tok;
                    #pragma unroll
                    for (int k = 0; k < KK; k++) {
                        uint32_t f[4];
                        vfrag(k, f);
                        f[0] &= k0;
                        f[1] &= k0;
                        f[2] &= k1;
                        f[3] &= k1;
                        float e4[4] = {0.f, 0.f, 0.f, 0.f};
                        mma8(e4, f, ph0, ph1);
                        mma8(e4, f, pw0, pw1);
                        if (c0) o[k][0] += e4[0];
                        if (c1) o[k][1] += e4[1];
                        if (c0) o[k][2] += e4[2];
                        if (c1) o[k][3] += e4[3];
                    }
                }
            }
            release();
        }
        // the sums of a row lie in the lanes of its column
        #pragma unroll
        for (int i = 0; i < 2; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
        }
        if (g == 0) {
            s_m[warp][2 * q4] = m[0];
            s_m[warp][2 * q4 + 1] = m[1];
            s_l[warp][2 * q4] = l[0];
            s_l[warp][2 * q4 + 1] = l[1];
        }
        if (!ok) {
            // a wait ran out: the copies still in flight land (bounded) before shared memory is given up
            for (; done < issued; done++) {
                mbar_wait_drain(bar0 + 8 * entry, (phase >> entry) & 1u, &g_status_paged);
                phase ^= 1u << entry;
                entry = entry + 1 == C::NST ? 0 : entry + 1;
            }
        }
        // the ring is empty now: it takes the warp's partial
        float* mine = reinterpret_cast<float*>(ring_p);
        #pragma unroll
        for (int k = 0; k < KK; k++) {
            mine[(2 * q4) * C::PITCH + 16 * k + g] = o[k][0];
            mine[(2 * q4 + 1) * C::PITCH + 16 * k + g] = o[k][1];
            mine[(2 * q4) * C::PITCH + 16 * k + g + 8] = o[k][2];
            mine[(2 * q4 + 1) * C::PITCH + 16 * k + g + 8] = o[k][3];
        }
        __syncthreads();
        if (*abort) break;                       // the same for the whole CTA: it is set before the barrier only
        const bool whole = nu == t.n;
        const bool direct = whole && t.solo;
        const float* parts = reinterpret_cast<const float*>(ring_p - warp * C::NST * C::ENTRY);
        constexpr int WP = C::NST * C::ENTRY / 4;    // floats between two warps' partials
        for (int e = tid; e < t.nrows * (HD / 4); e += 32 * kFewWarps) {
            const int r = e / (HD / 4), c = 4 * (e % (HD / 4));
            float M = s_m[0][r];
            #pragma unroll
            for (int w = 1; w < kFewWarps; w++) M = fmaxf(M, s_m[w][r]);
            const float mu = M == -INFINITY ? 0.f : M;
            float L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
            #pragma unroll
            for (int w = 0; w < kFewWarps; w++) {
                const float f = exp2_approx(s_m[w][r] - mu) * kFewDrop;
                L = fmaf(s_l[w][r], f, L);
                const float4 p = *reinterpret_cast<const float4*>(parts + w * WP + r * C::PITCH + c);
                v[0] = fmaf(p.x, f, v[0]);
                v[1] = fmaf(p.y, f, v[1]);
                v[2] = fmaf(p.z, f, v[2]);
                v[3] = fmaf(p.w, f, v[3]);
            }
            const int row = t.row0 + r, tok = row / G, hq = head * G + row % G;
            if (direct) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                const long long at0 = (long long)tok * a.out_stride + (long long)hq * HD + c;
                if (a.out_f32) {
                    *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at0) =
                        make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                } else {
                    uint2 p;
                    p.x = half_pair(v[0] * inv, v[1] * inv);
                    p.y = half_pair(v[2] * inv, v[3] * inv);
                    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(a.out) + at0) = p;
                }
            } else {
                // whole: the row's own slot; else this CTA's edge slot: 1 for the tile's first piece, 0 for a later
                const size_t slot = whole ? ((size_t)(t.seq < 0 ? 0 : 1) * d.T + tok) * d.nH + hq
                                          : ((size_t)blockIdx.x * 2 + (unit == 0 ? 1 : 0)) * kRowsS + r;
                float* dst = (whole ? a.w.row : a.w.edge[0]) + slot * HD + c;
                *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
                if (c == 0) *(whole ? a.w.row_ml + 2 * slot : a.w.edge_ml[0] + slot) = make_float2(M, L);
            }
        }
        // the ring was written and read by threads; the next piece's copies come behind that
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        left -= nu;
        unit += nu;
        if (unit == t.n) {
            left -= t.idle;
            unit = 0;
            ti++;
        }
    }
    // the join reads what this grid and the one before it wrote: done only when that one is
    pdl_wait();
}

// ------------------------------------------------------------------ join
// out = sum_p V_p 2^(m_p - M) / sum_p l_p 2^(m_p - M) over the partials of a row's prefix tile and of its own tile, for
// the rows that no whole tile wrote; a row with no key at all becomes zeros.  The plan lists groups of rows of a (tile,
// KV head) pair; a CTA takes a group at a time.  Where it has fewer rows than warps, several warps share a row's partials:
// a decode token over a long prefix has twenty or so, and their loads are what takes time here.

template <int HD>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Args a) {
    constexpr int PER = HD / 32;
    __shared__ float s_v[kJoinWarps][HD], s_m[kJoinWarps][32], s_l[kJoinWarps][32];
    const Dims& d = a.d;
    const Hdr* h = hdr_of(a.plan);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool fits = plan_fits(h, d);
    const int n0 = fits ? h->nj[0] : 0, items = n0 + (fits ? h->nj[1] : 0);
    bool waited = false;
    for (int it = blockIdx.x; it < items; it += gridDim.x) {
        // the plan's part first: no kernel before this one writes it
        const int kind = it >= n0, most = h->rj[kind];
        const int2 entry = at<int2>(a.plan, d.joins[kind])[kind ? it - n0 : it];
        const Tile t = at<Tile>(a.plan, d.tiles[kind])[entry.x];
        const int head = entry.y & 0xffff, row_a = (entry.y >> 16) * most, rows = min(most, t.nrows - row_a);
        const int share = rows > 4 ? 1 : rows > 2 ? 2 : rows > 1 ? 4 : 8;       // warps per row
        const int r = row_a + warp / share;
        const bool busy = r < t.nrows && warp / share < rows;
        const int row = t.row0 + min(r, t.nrows - 1), tok = row / d.G, hq = head * d.G + row % d.G;
        // A many-rows tile of a wide head is walked once per part of the columns; this lane's part may have been cut
        // elsewhere than another lane's.
        const float* part[2] = {nullptr, nullptr};      // of the prefix (0) and this tile (1): the first partial's sums,
        const float2* ml[2] = {nullptr, nullptr};       // its (maximum, sum),
        int n[2] = {0, 0}, next[2] = {0, 0}, width[2] = {HD, HD};   // how many; slots between later ones; floats of a slot
        bool done = false;
        #pragma unroll
        for (int seg = 0; seg < 2; seg++) {
            const int ref = seg ? 0 : __ldg(at<int>(a.plan, d.row_pre) + row);
            if (ref == -1) continue;
            const int k = seg ? kind : (unsigned)ref >> 31;
            const Tile& x = seg ? t : at<Tile>(a.plan, d.tiles[k])[ref & 0x7fffffff];
            if (x.n == 0) continue;
            width[seg] = k ? HD / d.cs : HD;
            const int walk = lane * PER / width[seg];
            const Span sp = span_of(h, k, x.off, x.n, k ? head * d.cs + walk : head);
            n[seg] = sp.c1 - sp.c0 + 1;
            if (sp.c0 == sp.c1) {
                done = x.solo;                          // these columns are written
                const size_t slot = ((size_t)seg * d.T + tok) * d.nH + hq;
                part[seg] = a.w.row + slot * HD + lane * PER;
                ml[seg] = a.w.row_ml + 2 * slot + walk;
            } else {
                // edge slots: 1 in the tile's first CTA, 0 in the ones behind it
                const int br = k ? kRowsP : kRowsS;
                const size_t slot = ((size_t)sp.c0 * 2 + 1) * br + (row - x.row0);
                part[seg] = a.w.edge[k] + slot * width[seg] + lane * PER % width[seg];
                ml[seg] = a.w.edge_ml[k] + slot;
                next[seg] = 2 * br;
            }
        }
        if (!waited) pdl_wait();
        waited = true;
        float M = -INFINITY, L = 0.f, v[PER];
        #pragma unroll
        for (int i = 0; i < PER; i++) v[i] = 0.f;
        const int total = busy && !done ? n[0] + n[1] : 0;
        constexpr int NB = HD == 512 ? 2 : 4;           // partials at once: their loads are independent, their sums are not
        for (int k0 = warp % share; k0 < total; k0 += NB * share) {
            float2 w2[NB];
            float x[NB][PER];
            #pragma unroll
            for (int k = 0; k < NB; k++) {
                const int p = k0 + k * share;
                w2[k] = make_float2(-INFINITY, 0.f);
                #pragma unroll
                for (int i = 0; i < PER; i++) x[k][i] = 0.f;
                if (p < total) {
                    const bool own = p >= n[0];
                    const int q = own ? p - n[0] : p;
                    // slots from the first partial: partial q > 0 is q pairs of slots on, less one
                    const long long s = q == 0 ? 0 : (long long)q * (own ? next[1] : next[0]) - (own ? next[1] : next[0]) / 2;
                    w2[k] = __ldcg((own ? ml[1] : ml[0]) + s);
                    const float* src = (own ? part[1] : part[0]) + s * (own ? width[1] : width[0]);
                    #pragma unroll
                    for (int i = 0; i < PER; i += 4) {
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(src + i));
                        x[k][i] = y.x;
                        x[k][i + 1] = y.y;
                        x[k][i + 2] = y.z;
                        x[k][i + 3] = y.w;
                    }
                }
            }
            float mn = M;
            #pragma unroll
            for (int k = 0; k < NB; k++) mn = fmaxf(mn, w2[k].x);
            const float mu = mn == -INFINITY ? 0.f : mn;
            const float f = exp2_approx(M - mu);
            M = mn;
            L *= f;
            #pragma unroll
            for (int i = 0; i < PER; i++) v[i] *= f;
            #pragma unroll
            for (int k = 0; k < NB; k++) {
                const float g = exp2_approx(w2[k].x - mu);
                L = fmaf(w2[k].y, g, L);
                #pragma unroll
                for (int i = 0; i < PER; i++) v[i] = fmaf(x[k][i], g, v[i]);
            }
        }
        if (share > 1) {
            // the row's warps add up; the first of them goes on
            #pragma unroll
            for (int i = 0; i < PER; i++) s_v[warp][lane + 32 * i] = v[i];
            s_m[warp][lane] = M;
            s_l[warp][lane] = L;
            __syncthreads();
            if (warp % share == 0) {
                for (int k = 1; k < share; k++) {
                    const float m2 = s_m[warp + k][lane], mn = fmaxf(M, m2), mu = mn == -INFINITY ? 0.f : mn;
                    const float f = exp2_approx(M - mu), g = exp2_approx(m2 - mu);
                    M = mn;
                    L = L * f + s_l[warp + k][lane] * g;
                    #pragma unroll
                    for (int i = 0; i < PER; i++) v[i] = v[i] * f + s_v[warp + k][lane + 32 * i] * g;
                }
            }
            __syncthreads();
        }
        if (!busy || done || warp % share != 0) continue;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const long long o = (long long)tok * a.out_stride + (long long)hq * HD + lane * PER;
        #pragma unroll
        for (int i = 0; i < PER; i++) v[i] *= inv;
        if (a.out_f32) {
            #pragma unroll
            for (int i = 0; i < PER; i += 4)
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + o + i) =
                    make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
            store_half<PER>(reinterpret_cast<uint16_t*>(a.out) + o, v);
        }
    }
    if (!waited) pdl_wait();    // a grid that ends is taken for the end of the one it depends on, too
}

// a launch that may begin while the kernel before it in the stream finishes
template <typename K, typename... A>
static cudaError_t launch_pdl(K k, dim3 grid, int threads, size_t smem, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

template <int HD>
static cudaError_t launch_few(const Args& a, const CUtensorMap& km, const CUtensorMap& vm, bool after_many,
                              cudaStream_t s) {
    using C = FewCfg<HD>;
    cudaError_t e = cudaFuncSetAttribute(few_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    // Behind the many-rows kernel its CTAs may begin as that one's end: they read nothing of it, and what both read was
    // complete before that one began (it is an ordinary launch).  Each waits for it before it ends.
    if (after_many) {
        e = launch_pdl(few_kernel<HD>, dim3(a.d.ctas[0]), 32 * kFewWarps, C::SMEM, s, a, km, vm);
    } else {
        few_kernel<HD><<<a.d.ctas[0], 32 * kFewWarps, C::SMEM, s>>>(a, km, vm);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) return e;
    const int most = a.d.T * a.d.nH;      // a group has a row at least
    return launch_pdl(join_kernel<HD>, dim3((unsigned)std::min(most, a.d.join_ctas)), kJoinThreads, 0, s, a);
}

template <int HD, bool XF32>
static cudaError_t launch_append_hd(const AppendArgs& a, int sms, cudaStream_t s) {
    const int heads = a.d.nH + 2 * a.d.nkv, per = kAppendThreads / 32;
    const int bytes = stage_bytes(a.d, XF32 ? 4 : 2);
    // As many stages as the ring holds; a token too wide for two stages takes the other kernel.  So do tokens with fewer
    // heads than this kernel has head warps, some of which would stand idle (8 / 1 heads of 128, 9,472 tokens: 27.0 us
    // against 23.4; 4 / 2 of 256, 4,736: 17.7 against 15.2), and batches of few elements: the two are level at 3 to 7 M
    // (16 / 8 heads of 256, f16: 444 tokens 7.6 us against 6.7, 592 8.0 against 8.7, 1,184 12.4 against 15.2; 8 / 8 of
    // 128: 1,184 tokens 7.6 against 7.5, 2,368 12.5 against 13.5; 16 / 1 of 512: 296 tokens 8.7 against 8.9, 1,184 18.1
    // against 26.1; 4 / 2 of 512: 1,184 tokens 12.6 against 11.5, 3,832 25.8 against 31.5).
    const int stages = std::min(8, kStreamSmem / bytes);
    if (stages >= 2 && heads >= stream_warps(HD) && (long long)a.d.T * heads * HD >= 1 << 22) {
        cudaError_t e = cudaFuncSetAttribute(append_stream_kernel<HD, XF32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kStreamSmem);
        if (e != cudaSuccess) return e;
        append_stream_kernel<HD, XF32><<<2 * sms, 32 * (stream_warps(HD) + 1), stages * bytes, s>>>(a, stages);
    } else {
        append_kernel<HD, XF32><<<dim3(a.d.T, (heads + per - 1) / per), kAppendThreads, 0, s>>>(a);
    }
    return cudaGetLastError();
}

template <bool XF32>
static cudaError_t launch_append(const AppendArgs& a, int sms, cudaStream_t s) {
    return a.d.hd == 128 ? launch_append_hd<128, XF32>(a, sms, s)
         : a.d.hd == 256 ? launch_append_hd<256, XF32>(a, sms, s)
                         : launch_append_hd<512, XF32>(a, sms, s);
}

}  // namespace pg

unsigned read_status_paged() {
    const unsigned m = pg::read_status_paged_mma();
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, pg::g_status_paged, sizeof(v)) != cudaSuccess) return 0xffffffffu;
    if (v) {
        const unsigned zero = 0;
        cudaMemcpyToSymbol(pg::g_status_paged, &zero, sizeof(zero));
    }
    return v | m;
}

}  // namespace g4b

using namespace g4b;
using namespace g4b::pg;

extern "C" {

size_t g4b_paged_plan_bytes(int T, int B, int nH, int nkv, int hd, int page_size, int table_pages, int prefix_pages,
                            int window) {
    Dims d;
    clear_error();
    return make_dims("paged_plan_bytes", T, B, nH, nkv, hd, page_size, table_pages, prefix_pages, window, d) == G4B_OK
               ? d.bytes
               : 0;
}

size_t g4b_paged_workspace_bytes(int T, int B, int nH, int nkv, int hd, int page_size, int table_pages,
                                 int prefix_pages, int window) {
    Dims d;
    clear_error();
    return make_dims("paged_workspace_bytes", T, B, nH, nkv, hd, page_size, table_pages, prefix_pages, window, d) ==
                   G4B_OK
               ? work_bytes(d, nullptr, nullptr)
               : 0;
}

int g4b_paged_plan(const int* q_start, const int* kv_len, const int* prefix_len, int T, int B, int nH, int nkv, int hd,
                   int page_size, int table_pages, int prefix_pages, int window, void* plan, size_t plan_bytes,
                   g4b_stream_t stream) {
    G4B_ENTRY("paged_plan");
    G4B_REQUIRE(q_start && kv_len && plan, G4B_E_ARG, "paged_plan: NULL pointer");
    G4B_REQUIRE(prefix_pages == 0 || prefix_len, G4B_E_ARG, "paged_plan: %d prefix pages without prefix_len",
                prefix_pages);
    PlanArgs a{};
    int st = make_dims("paged_plan", T, B, nH, nkv, hd, page_size, table_pages, prefix_pages, window, a.d);
    if (st != G4B_OK) return st;
    G4B_REQUIRE(aligned16(plan), G4B_E_ALIGN, "paged_plan: the plan must be 16-byte aligned");
    G4B_REQUIRE(plan_bytes >= a.d.bytes, G4B_E_WORKSPACE, "paged_plan: needs %zu bytes, got %zu", a.d.bytes,
                plan_bytes);
    st = check_device(nullptr);
    if (st != G4B_OK) return st;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.prefix_len = prefix_pages > 0 ? prefix_len : nullptr;
    a.plan = plan;
    // (the limit is the same for every call: another thread's may come between it and the launch)
    const int smem = (3 * B + 1) * 4;
    cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * kMaxSeqs + 1) * 4);
    if (e != cudaSuccess) return fail(G4B_E_CUDA, "paged_plan: %s", cudaGetErrorString(e));
    const int rows = T * a.d.G;
    const int grid = std::min(64, (rows + 4 * kPlanThreads - 1) / (4 * kPlanThreads));
    plan_kernel<<<grid, kPlanThreads, smem, reinterpret_cast<cudaStream_t>(stream)>>>(a);
    count_launch();
    return launch_status("paged_plan");
}

int g4b_paged_append(const void* qkv, int dtype, long long row_stride, const float* qnw, const float* knw,
                     const float* cos_tab, const float* sin_tab, int n_pos, uint16_t* kc, uint16_t* vc, int num_pages,
                     const int* table, uint16_t* q_out, long long q_stride, int T, int B, int nH, int nkv, int hd,
                     int koff, int voff, int page_size, int table_pages, int prefix_pages, int window,
                     const void* plan, g4b_stream_t stream) {
    G4B_ENTRY("paged_append");
    G4B_REQUIRE(qkv && qnw && knw && cos_tab && sin_tab && kc && vc && table && q_out && plan, G4B_E_ARG,
                "paged_append: NULL pointer");
    G4B_REQUIRE(dtype == G4B_DT_F32 || dtype == G4B_DT_F16, G4B_E_ARG, "paged_append: bad dtype %d", dtype);
    AppendArgs a{};
    int st = make_dims("paged_append", T, B, nH, nkv, hd, page_size, table_pages, prefix_pages, window, a.d);
    if (st != G4B_OK) return st;
    G4B_REQUIRE(num_pages >= 1 && (long long)num_pages * nkv * page_size <= 0x7fff0000LL, G4B_E_SHAPE,
                "paged_append: %d pages of %d rows of %d heads", num_pages, page_size, nkv);
    G4B_REQUIRE(n_pos >= (table_pages + prefix_pages) * page_size, G4B_E_SHAPE,
                "paged_append: rotations of %d positions, the tables hold %d", n_pos,
                (table_pages + prefix_pages) * page_size);
    G4B_REQUIRE(koff >= 0 && voff >= 0 && koff % 8 == 0 && voff % 8 == 0 && row_stride % 8 == 0 && q_stride % 8 == 0 &&
                    q_stride >= (long long)nH * hd && row_stride >= (long long)nH * hd &&
                    row_stride >= (long long)koff + (long long)nkv * hd && row_stride >= (long long)voff + (long long)nkv * hd,
                G4B_E_SHAPE, "paged_append: row_stride=%lld q_stride=%lld koff=%d voff=%d (multiples of 8, rows inside)",
                row_stride, q_stride, koff, voff);
    G4B_REQUIRE(aligned16(qkv) && aligned16(qnw) && aligned16(knw) && aligned16(cos_tab) && aligned16(sin_tab) &&
                    aligned16(kc) && aligned16(vc) && aligned16(q_out) && aligned16(plan),
                G4B_E_ALIGN, "paged_append: qkv, the weights, the rotations, the caches, q_out and the plan must be "
                "16-byte aligned");
    const size_t cache = (size_t)num_pages * nkv * page_size * hd * 2, esz = dtype == G4B_DT_F32 ? 4 : 2;
    const long long last = std::max((long long)nH * hd, std::max(koff, voff) + (long long)nkv * hd);
    const Rows in{qkv, T, row_stride * (long long)esz, last * (long long)esz}, q{q_out, T, q_stride * 2, (long long)nH * hd * 2};
    G4B_REQUIRE(!rows_overlap(flat(kc, cache), flat(vc, cache)) && !rows_overlap(q, in) &&
                    !rows_overlap(q, flat(kc, cache)) && !rows_overlap(q, flat(vc, cache)) &&
                    !rows_overlap(in, flat(kc, cache)) && !rows_overlap(in, flat(vc, cache)),
                G4B_E_ARG, "paged_append: kc, vc, q_out and qkv overlap");
    a.plan = plan;
    a.qkv = qkv;
    a.qnw = qnw;
    a.knw = knw;
    a.cos_t = cos_tab;
    a.sin_t = sin_tab;
    a.kc = kc;
    a.vc = vc;
    a.table = table;
    a.q_out = q_out;
    a.row_stride = row_stride;
    a.q_stride = q_stride;
    a.koff = koff;
    a.voff = voff;
    a.num_pages = num_pages;
    int sms = 148;
    st = check_device(&sms);
    if (st != G4B_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == G4B_DT_F32 ? launch_append<true>(a, sms, s) : launch_append<false>(a, sms, s);
    if (e != cudaSuccess) return fail(G4B_E_CUDA, "paged_append: launch: %s", cudaGetErrorString(e));
    count_launch();
    return launch_status("paged_append");
}

int g4b_paged_attn(const uint16_t* q, long long q_stride, const uint16_t* kc, const uint16_t* vc, int num_pages,
                   const int* table, const int* prefix_table, void* out, int out_dtype, long long out_stride,
                   float scale, int T, int B, int nH, int nkv, int hd, int page_size, int table_pages,
                   int prefix_pages, int window, const void* plan, void* workspace, size_t ws_bytes,
                   g4b_stream_t stream) {
    G4B_ENTRY("paged_attn");
    G4B_REQUIRE(q && kc && vc && table && out && plan, G4B_E_ARG, "paged_attn: NULL pointer");
    G4B_REQUIRE(prefix_pages == 0 || prefix_table, G4B_E_ARG, "paged_attn: %d prefix pages without prefix_table",
                prefix_pages);
    G4B_REQUIRE(out_dtype == G4B_DT_F32 || out_dtype == G4B_DT_F16, G4B_E_ARG, "paged_attn: bad out_dtype %d",
                out_dtype);
    G4B_REQUIRE(scale > 0.f && scale < 1e30f, G4B_E_ARG, "paged_attn: scale=%g (positive and finite)", (double)scale);
    Args a{};
    int st = make_dims("paged_attn", T, B, nH, nkv, hd, page_size, table_pages, prefix_pages, window, a.d);
    if (st != G4B_OK) return st;
    G4B_REQUIRE(num_pages >= 1 && (long long)num_pages * nkv * page_size <= 0x7fff0000LL, G4B_E_SHAPE,
                "paged_attn: %d pages of %d rows of %d heads", num_pages, page_size, nkv);
    G4B_REQUIRE(q_stride >= (long long)nH * hd && out_stride >= (long long)nH * hd && q_stride % 8 == 0 &&
                    out_stride % 8 == 0,
                G4B_E_SHAPE, "paged_attn: q_stride=%lld out_stride=%lld (multiples of 8, >= nH * hd)", q_stride,
                out_stride);
    G4B_REQUIRE(aligned16(q) && aligned16(kc) && aligned16(vc) && aligned16(out) && aligned16(plan), G4B_E_ALIGN,
                "paged_attn: q, the caches, out and the plan must be 16-byte aligned");
    const size_t need = work_bytes(a.d, nullptr, nullptr);
    G4B_REQUIRE(workspace && aligned16(workspace) && ws_bytes >= need, G4B_E_WORKSPACE,
                "paged_attn: needs a 16-byte aligned workspace of %zu bytes, got %zu", need, ws_bytes);
    const size_t cache = (size_t)num_pages * nkv * page_size * hd * 2, osz = out_dtype == G4B_DT_F32 ? 4 : 2;
    const long long wide = (long long)nH * hd;
    const Rows to{out, T, out_stride * (long long)osz, wide * (long long)osz};
    G4B_REQUIRE(!rows_overlap(to, Rows{q, T, q_stride * 2, wide * 2}) && !rows_overlap(to, flat(kc, cache)) &&
                    !rows_overlap(to, flat(vc, cache)),
                G4B_E_ARG, "paged_attn: out overlaps q or the caches");
    work_bytes(a.d, reinterpret_cast<char*>(workspace), &a.w);
    a.plan = plan;
    a.q = q;
    a.kc = kc;
    a.vc = vc;
    a.table = table;
    a.pre_table = prefix_table;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.scale = scale * 1.4426950408889634f;
    a.out_f32 = out_dtype == G4B_DT_F32;
    a.num_pages = num_pages;
    st = check_device(nullptr);
    if (st != G4B_OK) return st;
    CUtensorMap km, vm;
    const uint64_t rows = (uint64_t)num_pages * nkv * page_size;
    for (int i = 0; i < 2; i++) {
        st = tensor_map_chunks(i ? &vm : &km, i ? vc : kc, hd, rows, kBlk, hd / 64);
        if (st != G4B_OK) return st;
    }
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    // no tile of many rows: neither a sequence nor the prefix has more rows than the batch
    const bool many = T * a.d.G > a.d.few;
    if (many) {
        st = launch_many(a, s);
        if (st != G4B_OK) return st;
    }
    cudaError_t e = hd == 128 ? launch_few<128>(a, km, vm, many, s)
                  : hd == 256 ? launch_few<256>(a, km, vm, many, s)
                              : launch_few<512>(a, km, vm, many, s);
    if (e != cudaSuccess) return fail(G4B_E_CUDA, "paged_attn: launch: %s", cudaGetErrorString(e));
    count_launch(2);
    return launch_status("paged_attn");
}

}  // extern "C"
