// g4b_paged_mma.cu -- attention over the paged cache where many rows share the keys: a prefix read for all
// sequences at once, and the chunks of prompts.
//
// A tile is 128 rows (token, query head of the group) of one KV head, a row per tensor memory lane; units of 64
// keys stream past it.  Per unit
//   S [128 x 64] = Q K^T      (tcgen05, Q in tensor memory, K from shared memory)
//   P = 2^(S scale - m)       (one thread per row: no reduction leaves the thread)
//   O [128 x hd] += P V       (tcgen05, P in tensor memory over S's columns, V from shared memory)
// S is double buffered, so the tensor core makes unit i + 1's scores while the softmax warps work on unit i.
// m is the maximum seen when it was last set: O is rescaled only where a row's maximum has risen by more than
// 2^8 since (weights up to 256 are exact enough in f16: their relative rounding does not change).
// K and V units come by TMA through one ring of 64-key buffers, issued ahead across pieces.
//
// Warps: 0-3 softmax, the mask, the rows' Q and the result; 4 TMA; 5 MMA issue.
// At hd 512 the 512 output columns of O would fill tensor memory, so a tile is walked once for each half of
// them (the scores are made twice), and half of Q stays in shared memory.
//
// The weights P are rounded to f16, the type of V, as the tensor core needs one type for both: 2^-11 of each
// weight, unbiased; sums and maxima are f32.
#include "g4b_paged.cuh"
#include "g4b_tcgen05.cuh"

namespace g4b {
namespace pg {

__device__ unsigned g_status_paged_mma;

constexpr int kManyThreads = 192;
constexpr int kPieceRowsMin = 16;       // smallest page: rows of a TMA box
constexpr float kLazy = 8.f;            // log2 of how far weights may rise before O is rescaled

template <int HD>
struct ManyCfg {
    static constexpr int DV = HD < 256 ? HD : 256;      // output columns of a walk
    static constexpr int CS = HD / DV;                  // walks per tile
    static constexpr int QT = DV;                       // elements of Q in tensor memory; the rest in shared memory
    static constexpr int KE = HD / QT;                  // ring entries per unit of K
    static constexpr int ENTRY = kUnit * DV * 2;        // bytes of a ring entry: 64 keys x DV elements
    static constexpr int QS_BYTES = kRowsP * (HD - QT) * 2;
    static constexpr int NST = HD == 128 ? 12 : HD == 256 ? 7 : 5;
    static constexpr int SMEM = NST * ENTRY + QS_BYTES + 1024;
    static constexpr int O_COL = 0, S_COL = DV, Q_COL = DV + 2 * kUnit;
    static_assert(Q_COL + QT / 2 <= 512, "tensor memory columns");
    static_assert(SMEM <= 226 * 1024, "shared memory");
    static_assert(KE * 2 + 1 <= NST, "the units issued before the first release");
};

namespace {

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ uint32_t ld_tmem_x1(uint32_t taddr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr) : "memory");
    return v;
}

// The pieces of a CTA's stretch, walked alike by every role.
struct Walk {
    const Tile* tiles;
    long long left;
    int ntiles, head, ti, unit;   // head: KV head * CS + column part
    Tile t;
    int nu, key0, key1;

    __device__ __forceinline__ bool init(const Args& a) {
        const Hdr* h = hdr_of(a.plan);
        const Start st = at<Start>(a.plan, a.d.start[1])[blockIdx.x];
        if (st.head < 0) return false;
        tiles = at<Tile>(a.plan, a.d.tiles[1]);
        ntiles = h->nt[1];
        head = st.head;
        ti = st.tile;
        unit = st.unit;
        left = min(h->u[1], h->wt[1] * a.d.nkv * a.d.cs - (long long)blockIdx.x * h->u[1]);
        return true;
    }
    __device__ __forceinline__ bool next() {
        while (left > 0) {
            if (ti == ntiles) {
                ti = 0;
                head++;
            }
            t = tiles[ti];
            if (t.n > 0) break;
            ti++;
            unit = 0;
        }
        if (left <= 0) return false;
        nu = (int)min((long long)(t.n - unit), left);
        key0 = t.lo + unit * kUnit;
        key1 = min(t.hi, key0 + nu * kUnit);
        return true;
    }
    __device__ __forceinline__ void step() {
        left -= nu;
        unit += nu;
        if (unit == t.n) {
            unit = 0;
            ti++;
        }
    }
};

}  // namespace

template <int HD>
__global__ void __launch_bounds__(kManyThreads, 1)
many_kernel(const Args a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using C = ManyCfg<HD>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * C::NST + 8];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_acc, s_red[4][4];
    __shared__ unsigned long long s_odd;         // keys of the unit with a value that is not finite
    const Dims& d = a.d;
    const Hdr* h = hdr_of(a.plan);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // The next kernel may begin: it reads nothing of this one, and waits for its end before it ends itself.
    pdl_launch_dependents();
    if (h->sig != d.sig) {
        if (blockIdx.x == 0 && tid == 0) atomicOr(&g_status_paged_mma, kStatusPlan);
        return;
    }
    Walk w;
    if (!w.init(a)) return;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* ring_p = smem_raw + (ring - smem_u32(smem_raw));
    const uint32_t qs = ring + C::NST * C::ENTRY;                    // hd 512: the second half of Q
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (C::NST + s); };
    const uint32_t b_s = bar0 + 8u * (2 * C::NST);                   // [2] scores of a unit are there
    const uint32_t b_p = b_s + 16;                                   // [2] its weights are there
    const uint32_t b_pv = b_s + 32;                                  // [2] its product is added
    const uint32_t b_q = b_s + 48;                                   // the piece's Q is there
    const uint32_t b_drain = b_s + 56;
    if (tid == 0) {
        for (int i = 0; i < 2 * C::NST; i++) mbar_init(bar0 + 8u * i, 1);
        mbar_init(b_s, 1);
        mbar_init(b_s + 8, 1);
        mbar_init(b_p, 128);
        mbar_init(b_p + 8, 128);
        mbar_init(b_pv, 1);
        mbar_init(b_pv + 8, 1);
        mbar_init(b_q, 128);
        mbar_init(b_drain, 1);
        fence_mbar_init();
        s_abort = 0;
    }
    if (warp == 5) {
        tc::tmem_alloc(smem_u32(&s_tmem), 512);
        tc::tmem_relinquish();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = s_tmem;
    volatile int* abort = &s_abort;
    unsigned* status = &g_status_paged_mma;
    const int pl = h->prefix_len, G = d.G;

    if (warp == 4) {
        // ---------------------------------------------------------------- TMA
        long long e = 0;                          // entries issued
        bool ok = true;
        while (ok && w.next()) {
            const int head = w.head / C::CS, part = w.head % C::CS;
            const int* table = w.t.seq < 0 ? a.pre_table : a.table + (size_t)w.t.seq * d.own_pages;
            const int table_n = w.t.seq < 0 ? d.pre_pages : d.own_pages;
            const int box = min(d.ps, kUnit), boxes = kUnit / box;   // rows of a box, boxes per unit
            int ids = -1, ids_at = -64;
            // unit u of the piece: K (all of hd) or V (this walk's columns)
            auto load = [&](int u, bool is_v) {
                const int key = w.key0 + u * kUnit;
                int row[kUnit / kPieceRowsMin];
                #pragma unroll
                for (int p = 0; p < kUnit / kPieceRowsMin; p++) {
                    row[p] = 0;
                    if (p < boxes) {
                        const int k = key + p * box, idx = k / d.ps;
                        if (idx < ids_at || idx >= ids_at + 32) {
                            // 32 page ids ahead; from the unit before on, whose V may still be to come
                            ids_at = max(w.key0, key - kUnit) / d.ps;
                            ids = ids_at + lane < table_n ? __ldg(table + ids_at + lane) : -1;
                        }
                        const int id = __shfl_sync(0xffffffffu, ids, idx - ids_at);
                        const int r = cache_row(id, a.num_pages, d.nkv, d.ps, head, k);
                        row[p] = r < 0 ? a.num_pages * d.nkv * d.ps : r;   // past the map: zeros
                    }
                }
                for (int part_e = 0; part_e < (is_v ? 1 : C::KE); part_e++) {
                    const int s = (int)(e % C::NST);
                    const uint32_t use = (uint32_t)(e / C::NST);
                    if (use > 0 && !mbar_wait(empty(s), (use - 1) & 1u, abort, status)) ok = false;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) return;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(full(s), C::ENTRY);
                        const int x0 = (is_v ? part : part_e) * C::DV;
                        for (int c = 0; c < C::DV / 64; c++)
                            #pragma unroll
                            for (int p = 0; p < kUnit / kPieceRowsMin; p++)
                                if (p < boxes)
                                    tma_box(ring + s * C::ENTRY + c * (kUnit * 128) + p * box * 128, is_v ? &vmap : &kmap,
                                            x0 + 64 * c, row[p], full(s));
                    }
                    e++;
                }
            };
            load(0, false);
            for (int u = 0; u < w.nu && ok; u++) {
                if (u + 1 < w.nu) load(u + 1, false);
                if (ok) load(u, true);
            }
            w.step();
        }
        __syncwarp();
        // every copy lands before the CTA gives up its shared memory
        if (*abort)
            for (int s = 0; s < C::NST; s++) {
                const long long uses = e > s ? (e - s - 1) / C::NST + 1 : 0;
                if (uses > 0) mbar_wait_drain(full(s), (uint32_t)((uses - 1) & 1), status);
            }
    } else if (warp == 5) {
        // ---------------------------------------------------------------- MMA
        if (lane == 0) {
            constexpr uint32_t id_s = tc::idesc(1, 0, 0, 0, 0, kUnit, kRowsP);
            constexpr uint32_t id_o = tc::idesc(1, 0, 0, 0, 1, C::DV, kRowsP);
            long long e = 0;
            uint32_t it = 0, piece = 0;            // units and pieces so far
            bool ok = true;
            auto entry = [&](int& s) {             // the next entry, once it has landed
                s = (int)(e % C::NST);
                ok = ok && mbar_wait(full(s), (uint32_t)(e / C::NST) & 1u, abort, status);
                e++;
                return ok;
            };
            auto scores = [&](uint32_t i) {
                const uint32_t ds = tmem + C::S_COL + (i & 1u) * kUnit;
                #pragma unroll
                for (int pe = 0; pe < C::KE; pe++) {
                    int s;
                    if (!entry(s)) return;
                    tc::fence_after();
                    #pragma unroll
                    for (int k = 0; k < C::QT / 16; k++) {
                        const uint64_t bd = tc::sdesc_sw128(ring + s * C::ENTRY + (k / 4) * (kUnit * 128), 16, 1024) +
                                            (uint64_t)((k % 4) * 2);
                        if (pe == 0) {
                            tc::mma_f16_ts(ds, tmem + C::Q_COL + 8 * k, bd, id_s, k > 0);
                        } else {
                            const uint64_t ad = tc::sdesc_sw128(qs + (k / 4) * (kRowsP * 128), 16, 1024) +
                                                (uint64_t)((k % 4) * 2);
                            tc::mma_f16_ss(ds, ad, bd, id_s, 1);
                        }
                    }
                    tc::commit(empty(s));
                }
                tc::commit(b_s + 8u * (i & 1u));
            };
            while (ok && w.next()) {
                ok = mbar_wait(b_q, piece & 1u, abort, status);
                piece++;
                tc::fence_after();
                if (ok) scores(it);
                for (int u = 0; ok && u < w.nu; u++) {
                    if (u + 1 < w.nu) scores(it + 1);
                    ok = ok && mbar_wait(b_p + 8u * (it & 1u), (it >> 1) & 1u, abort, status);
                    int s;
                    if (!ok || !entry(s)) break;
                    tc::fence_after();
                    const int acc = u > 0 || *(volatile int*)&s_acc;
                    #pragma unroll
                    for (int k = 0; k < kUnit / 16; k++)
                        tc::mma_f16_ts(tmem + C::O_COL, tmem + C::S_COL + (it & 1u) * kUnit + 8 * k,
                                       tc::sdesc_sw128(ring + s * C::ENTRY + k * 2048, kUnit * 128, 1024), id_o,
                                       acc || k > 0);
                    tc::commit(empty(s));
                    tc::commit(b_pv + 8u * (it & 1u));
                    it++;
                }
                w.step();
            }
            if (*abort) {
                tc::commit(b_drain);
                mbar_wait_drain(b_drain, 0, status);
            }
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- softmax: thread = row
        const uint32_t tl = tmem + ((uint32_t)(warp * 32) << 16);    // this warp's lanes
        uint32_t it = 0;                          // units so far
        long long e0 = 0;                         // ring entries of the pieces before
        // A wait that ran out clears ok.  The warp then walks on without waiting, so that the four warps meet at
        // the same named barriers to the end; it writes no result.
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = __all_sync(0xffffffffu, ok && mbar_wait(bar, parity, abort, status));
        };
        // The product of a unit is added.  A parity tells a barrier's last two phases apart only: units alternate
        // between two barriers, and every unit u waits for unit u - 2's, so neither runs ahead unseen.
        auto wait_pv = [&](uint32_t unit) {
            wait(b_pv + 8u * (unit & 1u), (unit >> 1) & 1u);
            tc::fence_after();
        };
        while (w.next()) {
            const int head = w.head / C::CS, part = w.head % C::CS;
            const bool live = tid < w.t.nrows;
            const int row = w.t.row0 + min(tid, w.t.nrows - 1);
            const int tok = row / G, hq = head * G + row % G;
            // Q's row into tensor memory (two elements per column) and, past QT, shared memory
            {
                const uint4* src = reinterpret_cast<const uint4*>(a.q + (long long)tok * a.q_stride + (long long)hq * HD);
                #pragma unroll
                for (int c = 0; c < C::QT / 64; c++) {
                    uint32_t v[32];
                    #pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint4 x = live ? __ldg(src + c * 8 + j) : make_uint4(0, 0, 0, 0);
                        v[4 * j] = x.x;
                        v[4 * j + 1] = x.y;
                        v[4 * j + 2] = x.z;
                        v[4 * j + 3] = x.w;
                    }
                    tc::st_32x32b_x32(tl + C::Q_COL + 32 * c, v);
                }
                if constexpr (HD > C::QT) {
                    #pragma unroll 8
                    for (int j = 0; j < (HD - C::QT) / 8; j++) {
                        const uint4 x = live ? __ldg(src + C::QT / 8 + j) : make_uint4(0, 0, 0, 0);
                        const uint32_t dst = qs + (j / 8) * (kRowsP * 128) + tid * 128 + (((j & 7) ^ (tid & 7)) << 4);
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(x.x), "r"(x.y), "r"(x.z),
                                     "r"(x.w) : "memory");
                    }
                    tc::fence_proxy_async_smem();
                }
                tc::wait_st();
                tc::fence_before();
                mbar_arrive(b_q);
            }
            const int kbase = w.t.seq < 0 ? 0 : pl;
            const int* table = w.t.seq < 0 ? a.pre_table : a.table + (size_t)w.t.seq * d.own_pages;
            const int table_n = w.t.seq < 0 ? d.pre_pages : d.own_pages;
            const int pos = __ldg(at<int>(a.plan, d.tok_pos) + tok);
            const int vhi = min(w.key1, pos + 1 - kbase), vlo = d.window > 0 ? max(0, pos + 1 - d.window - kbase) : 0;
            // keys that all rows see, keys that any row sees
            int all_lo = __reduce_max_sync(0xffffffffu, vlo), all_hi = __reduce_min_sync(0xffffffffu, vhi);
            int any_lo = __reduce_min_sync(0xffffffffu, vlo), any_hi = __reduce_max_sync(0xffffffffu, vhi);
            named_bar_sync(1, 128);               // the piece before has been read out of s_red
            if (lane == 0) {
                s_red[warp][0] = all_lo;
                s_red[warp][1] = all_hi;
                s_red[warp][2] = any_lo;
                s_red[warp][3] = any_hi;
            }
            named_bar_sync(1, 128);
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                all_lo = max(all_lo, s_red[i][0]);
                all_hi = min(all_hi, s_red[i][1]);
                any_lo = min(any_lo, s_red[i][2]);
                any_hi = max(any_hi, s_red[i][3]);
            }
            // page ids of a unit, one per box, in the first lanes; fetched a unit ahead
            const int box = min(d.ps, kUnit), boxes = kUnit / box, lbox = __ffs(box) - 1;
            auto page_of = [&](int u) {
                const int k = w.key0 + u * kUnit + (lane & 3) * box, idx = k / d.ps;
                return lane < boxes && u < w.nu && idx < table_n ? __ldg(table + idx) : -1;
            };
            int page = page_of(0);
            float m = -INFINITY, l = 0.f;
            for (int u = 0; u < w.nu; u++, it++) {
                const int key = w.key0 + u * kUnit;
                const unsigned there = __ballot_sync(0xffffffffu, lane < boxes && page >= 0 && page < a.num_pages);
                page = page_of(u + 1);
                const bool edge = there != (1u << boxes) - 1 || key < all_lo || key + kUnit > all_hi;
                wait(b_s + 8u * (it & 1u), (it >> 1) & 1u);
                if (it >= 2) wait_pv(it - 2);
                tc::fence_after();
                const uint32_t ts = tl + C::S_COL + (it & 1u) * kUnit;
                uint32_t x0[32], x1[32];
                tc::ld_32x32b_x32(ts, x0);
                tc::ld_32x32b_x32(ts + 32, x1);
                tc::wait_ld();
                if (edge) {
                    #pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const bool ta = (there >> (j >> lbox)) & 1u, tb = (there >> ((j + 32) >> lbox)) & 1u;
                        if (!ta || key + j < vlo || key + j >= vhi) x0[j] = 0xff800000u;
                        if (!tb || key + j + 32 < vlo || key + j + 32 >= vhi) x1[j] = 0xff800000u;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                #pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    mx[0] = fmaxf(mx[0], __uint_as_float(x0[j]));
                    mx[1] = fmaxf(mx[1], __uint_as_float(x0[j + 1]));
                    mx[2] = fmaxf(mx[2], __uint_as_float(x1[j]));
                    mx[3] = fmaxf(mx[3], __uint_as_float(x1[j + 1]));
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale;
                // units so far of this piece are in O: rescale it where a row's maximum has left its base behind
                if (u == 0) {
                    m = top;
                } else {
                    const bool rise = top > m + kLazy || (m == -INFINITY && top > m);
                    if (__any_sync(0xffffffffu, rise)) {
                        const float f = rise ? exp2_approx(m - top) : 1.f;     // m = -inf: nothing was added yet
                        if (rise) m = top;
                        l *= f;
                        wait_pv(it - 1);
                        #pragma unroll
                        for (int c = 0; c < C::DV; c += 32) {
                            uint32_t o[32];
                            tc::ld_32x32b_x32(tl + C::O_COL + c, o);
                            tc::wait_ld();
                            #pragma unroll
                            for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            tc::st_32x32b_x32(tl + C::O_COL + c, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m;
                float sum[2] = {0.f, 0.f};
                uint32_t p[32];
                #pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float e00 = exp2_approx(fmaf(__uint_as_float(x0[2 * j]), a.scale, -base));
                    const float e01 = exp2_approx(fmaf(__uint_as_float(x0[2 * j + 1]), a.scale, -base));
                    const float e10 = exp2_approx(fmaf(__uint_as_float(x1[2 * j]), a.scale, -base));
                    const float e11 = exp2_approx(fmaf(__uint_as_float(x1[2 * j + 1]), a.scale, -base));
                    sum[0] += e00 + e01;
                    sum[1] += e10 + e11;
                    const __half2 h0 = __floats2half2_rn(e00, e01), h1 = __floats2half2_rn(e10, e11);
                    p[j] = *reinterpret_cast<const uint32_t*>(&h0);
                    p[16 + j] = *reinterpret_cast<const uint32_t*>(&h1);
                }
                l += sum[0] + sum[1];
                tc::st_32x32b_x32(ts, p);
                if (u == 0 && tid == 0) *(volatile int*)&s_acc = 0;
                if (edge) {
                    // Values that no row sees become zeros; values that only some rows see and that are not
                    // finite (0 x NaN is not 0) are added row by row here and then cleared.
                    const long long ev = e0 + (u + 1 < w.nu ? (long long)C::KE * (u + 2) + u : (long long)C::KE * w.nu + u);
                    const int s = (int)(ev % C::NST);
                    wait(full(s), (uint32_t)(ev / C::NST) & 1u);
                    if (tid == 0) s_odd = 0;
                    named_bar_sync(1, 128);
                    uint4* vt = reinterpret_cast<uint4*>(ring_p + s * C::ENTRY);    // [DV / 64][64 keys][8 x 16 bytes]
                    for (int i = tid; i < C::ENTRY / 16; i += 128) {
                        const int k = key + (i >> 3) % kUnit;
                        if (k < any_lo || k >= any_hi) {
                            vt[i] = make_uint4(0, 0, 0, 0);
                        } else if (k < all_lo || k >= all_hi) {
                            const uint4 v = vt[i];
                            auto odd = [](uint32_t y) {
                                return (y & 0x7c00u) == 0x7c00u || (y & 0x7c000000u) == 0x7c000000u;
                            };
                            if (odd(v.x) || odd(v.y) || odd(v.z) || odd(v.w))
                                atomicOr(&s_odd, 1ull << ((i >> 3) % kUnit));
                        }
                    }
                    named_bar_sync(1, 128);
                    unsigned long long odd = s_odd;
                    if (odd) {
                        tc::wait_st();                       // P, read back below
                        if (u > 0) {
                            wait_pv(it - 1);
                        } else {
                            uint32_t z[32];
                            #pragma unroll
                            for (int j = 0; j < 32; j++) z[j] = 0;
                            #pragma unroll
                            for (int c = 0; c < C::DV; c += 32) tc::st_32x32b_x32(tl + C::O_COL + c, z);
                            tc::wait_st();
                            if (tid == 0) *(volatile int*)&s_acc = 1;
                        }
                        while (odd) {
                            const int j = __ffsll((long long)odd) - 1;
                            odd &= odd - 1;
                            const uint32_t pj = ld_tmem_x1(ts + j / 2);
                            tc::wait_ld();
                            const float pf = j & 1 ? h_hi(pj) : h_lo(pj);
                            const bool sees = key + j >= vlo && key + j < vhi && ((there >> (j >> lbox)) & 1u);
                            #pragma unroll 1
                            for (int c = 0; c < C::DV; c += 32) {
                                uint32_t o[32];
                                tc::ld_32x32b_x32(tl + C::O_COL + c, o);
                                tc::wait_ld();
                                const uint8_t* vr = ring_p + s * C::ENTRY + (c / 64) * (kUnit * 128) + j * 128;
                                #pragma unroll
                                for (int q = 0; q < 4; q++) {
                                    const int un = (c % 64) / 8 + q;
                                    const uint4 v = *reinterpret_cast<const uint4*>(vr + ((un ^ (j & 7)) << 4));
                                    const uint32_t y[4] = {v.x, v.y, v.z, v.w};
                                    #pragma unroll
                                    for (int r = 0; r < 4; r++) {
                                        float lo = __uint_as_float(o[8 * q + 2 * r]), hi = __uint_as_float(o[8 * q + 2 * r + 1]);
                                        if (sees) {
                                            lo += pf * h_lo(y[r]);
                                            hi += pf * h_hi(y[r]);
                                        }
                                        o[8 * q + 2 * r] = __float_as_uint(lo);
                                        o[8 * q + 2 * r + 1] = __float_as_uint(hi);
                                    }
                                }
                                tc::st_32x32b_x32(tl + C::O_COL + c, o);
                                tc::wait_st();
                            }
                        }
                        named_bar_sync(1, 128);              // every row has read the values
                        odd = s_odd;
                        for (int i = tid; i < C::ENTRY / 16; i += 128)
                            if ((odd >> ((i >> 3) % kUnit)) & 1ull) vt[i] = make_uint4(0, 0, 0, 0);
                    }
                    tc::fence_proxy_async_smem();
                }
                tc::wait_st();
                tc::fence_before();
                mbar_arrive(b_p + 8u * (it & 1u));
            }
            wait_pv(it - 1);
            // the row's result: finished, or this stretch's part of it
            const bool whole = w.nu == w.t.n, direct = whole && w.t.solo;
            const float inv = !direct ? 1.f : l == 0.f ? 0.f : 1.f / l;
            const size_t slot = whole ? ((size_t)(w.t.seq < 0 ? 0 : 1) * d.T + tok) * d.nH + hq
                                      : ((size_t)blockIdx.x * 2 + (w.unit == 0 ? 1 : 0)) * kRowsP + tid;
            float* dst = whole ? a.w.row + slot * HD + part * C::DV : a.w.edge[1] + slot * C::DV;
            const long long at0 = (long long)tok * a.out_stride + (long long)hq * HD + part * C::DV;
            if (live && ok && !direct) {
                if (whole) a.w.row_ml[slot * 2 + part] = make_float2(m, l);
                else a.w.edge_ml[1][slot] = make_float2(m, l);
            }
            #pragma unroll 2
            for (int c = 0; c < C::DV; c += 32) {
                uint32_t o[32];
                tc::ld_32x32b_x32(tl + C::O_COL + c, o);
                tc::wait_ld();
                if (!live || !ok) continue;
                if (direct && !a.out_f32) {
                    uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<__half*>(a.out) + at0 + c);
                    #pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint32_t y[4];
                        #pragma unroll
                        for (int r = 0; r < 4; r++)
                            y[r] = pack_half2(__float2half_rn(__uint_as_float(o[8 * j + 2 * r]) * inv),
                                              __float2half_rn(__uint_as_float(o[8 * j + 2 * r + 1]) * inv));
                        out[j] = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                } else {
                    float4* out = reinterpret_cast<float4*>(direct ? reinterpret_cast<float*>(a.out) + at0 + c : dst + c);
                    #pragma unroll
                    for (int j = 0; j < 8; j++)
                        out[j] = make_float4(__uint_as_float(o[4 * j]) * inv, __uint_as_float(o[4 * j + 1]) * inv,
                                             __uint_as_float(o[4 * j + 2]) * inv, __uint_as_float(o[4 * j + 3]) * inv);
                }
            }
            tc::fence_before();
            e0 += (long long)(C::KE + 1) * w.nu;
            w.step();
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 5) tc::tmem_dealloc(tmem, 512);
}

bool many_rows(int hd) { return hd == 128 || hd == 256 || hd == 512; }

template <int HD>
static cudaError_t launch(const Args& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(many_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, ManyCfg<HD>::SMEM);
    if (e != cudaSuccess) return e;
    many_kernel<HD><<<a.d.ctas[1], kManyThreads, ManyCfg<HD>::SMEM, s>>>(a, km, vm);
    return cudaGetLastError();
}

int launch_many(const Args& a, cudaStream_t s) {
    CUtensorMap km, vm;
    const uint64_t rows = (uint64_t)a.num_pages * a.d.nkv * a.d.ps;
    for (int i = 0; i < 2; i++) {
        const int st = tensor_map_2d(i ? &vm : &km, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, i ? a.vc : a.kc, a.d.hd, rows,
                                     (uint64_t)a.d.hd * 2, 64, a.d.ps < kUnit ? a.d.ps : kUnit, CU_TENSOR_MAP_SWIZZLE_128B);
        if (st != G4B_OK) return st;
    }
    const cudaError_t e = a.d.hd == 128 ? launch<128>(a, km, vm, s)
                        : a.d.hd == 256 ? launch<256>(a, km, vm, s)
                                        : launch<512>(a, km, vm, s);
    if (e != cudaSuccess) return fail(G4B_E_CUDA, "paged_attn: launch: %s", cudaGetErrorString(e));
    count_launch();
    return G4B_OK;
}

unsigned read_status_paged_mma() {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_status_paged_mma, sizeof(v)) != cudaSuccess) return 0xffffffffu;
    if (v) {
        const unsigned zero = 0;
        cudaMemcpyToSymbol(g_status_paged_mma, &zero, sizeof(zero));
    }
    return v;
}

}  // namespace pg
}  // namespace g4b
