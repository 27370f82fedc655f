// g4b_paged_mma.cu -- attention over the paged cache where many rows share the keys: a prefix read for many
// sequences at once, and the chunks of prompts.
//
// A tile is 128 rows (token, query head of the group) of one KV head, a row per tensor memory lane; units of 64
// keys stream past it.  Per unit
//   S [128 x 64] = Q K^T      (tcgen05, Q in tensor memory, K from shared memory)
//   P = 2^(S scale - m)       (a thread per row: no reduction leaves it; two groups of four warps take units in turn)
//   O [128 x hd] += P V       (tcgen05, P in tensor memory over S's columns, V from shared memory)
// S is double buffered and P has columns of its own, so the tensor core makes the scores two units ahead: a buffer is
// free as soon as its scores have been read, and the softmax warps find the next ones ready.  (With P over S, the scores of
// unit i + 1 waited for the product of unit i - 1.)
// m is a base, 2^4 under the maximum seen when it was set: O is rescaled only where a row's weights would pass
// 2^15, the last power of two of f16 (a larger weight's relative rounding is the same; the 2^4 keep weights down
// to 2^-18 of the maximum out of f16's subnormals, a low part's down to 2^-7).
// K and V units come by TMA through a ring each, issued ahead across pieces.
//
// Warps: 0-7 softmax, the mask, the rows' Q and the result; 8 and 11 the copies of K and V; 9 and 10 the MMAs.
// Tensor memory's 512 columns: O 256, S 128, P 32 and the first 192 elements of Q (64 and 128 where P has two parts); its
// others are in shared memory.  At hd 512 O alone would fill them, so a tile is walked once for each half of the output
// columns (the scores are made twice).
//
// The tensor core needs one type for P and V, so the weights enter as f16.  For an f16 result as one: 2^-11 of each
// weight, at most what the result's own rounding is, and a row's sum is of the rounded weights, so that what they have in
// common cancels (the error against 64 bits is 1.11 to 1.13 times that of 32-bit weights with the result rounded to f16; with
// the sum of the unrounded ones 1.22 to 1.34 times).  For an f32 result as two, a high and a low part: 2^-22 of each
// weight, and 8 products a unit where there were 4 (2 prompts of 4,096 at hd 256 339 us instead of 277, at hd 128 150
// instead of 131).  Either way weights below 2^-29 of the largest that its row had seen when its base was set count as
// nothing.  Maxima, sums and accumulators are f32.
//
// What bounds it: neither the tensor core nor memory.  A unit takes 1,410 clocks at hd 256, of which the MMAs are 1,100
// (1,300 and 550 at hd 128): the product of a unit waits for its weights, whose place is free when the product before is
// done, and each such hand-over from warp to warp and back is 150 to 300 clocks.  Deeper or shallower rings change
// nothing.  Between two pieces pass 12,000 clocks at hd 256 (16,000 before Q's chunks came all at once): Q in, the masks,
// the result out.  Two prompts of 4,096 tokens over 16 heads of 256 (8 KV heads): 284 us, 0.58 of the measured bf16
// rate; of 128 (8 heads, 1 KV head): 129 us, 0.32.
#include "g4b_paged.cuh"
#include "g4b_tcgen05.cuh"

namespace g4b {
namespace pg {

__device__ unsigned g_status_paged_mma;

constexpr int kGroup = 128;             // softmax threads of a group: one per row
constexpr int kSoft = 2 * kGroup;       // two groups
constexpr int kManyThreads = kSoft + 128;   // and a warp each for K's copies, V's, the scores and the products
constexpr float kLift = 4.f;            // log2 of the weight that a row's maximum gets when its base is set
constexpr float kMost = 15.f;           // log2 of the largest weight before the base is set anew (f16: below 2^16)
// From a base of this size on, an f32 step is no longer small beside a weight's exponent, and the exact product in
// x scale - base may lie steps above its rounded maximum: it is rounded as that one was before the base is taken off.
constexpr float kFar = 4194304.f;

template <int HD, bool PAIR>
struct ManyCfg {
    static constexpr int DV = HD < 256 ? HD : 256;      // output columns of a walk
    static constexpr int CS = HD / DV;                  // walks per tile
    static constexpr int PC = PAIR ? 2 : 1;             // f16 parts of a weight
    // elements of Q in tensor memory; the rest in shared memory
    static constexpr int QT = HD == 128 || PAIR ? 128 : 192;
    // A ring entry is 64 keys of EC elements; a unit's K is KE of them and its V (a walk's columns) VE.  K and V have a
    // ring each: then the one warp that consumes a ring sees every phase of its barriers.
    static constexpr int EC = HD == 512 ? 128 : DV;
    static constexpr int KE = HD / EC, VE = DV / EC;
    static constexpr int ENTRY = kUnit * EC * 2;
    static constexpr int NK = HD == 128 ? 5 : HD == 256 ? 3 : PAIR ? 5 : 6, NV = HD == 128 ? 5 : HD == 256 ? 2 : 3;
    static constexpr int NST = NK + NV;
    static constexpr int QS_BYTES = kRowsP * (HD - QT) * 2;
    // a warp's 32 rows x 128 bytes on their way between rows in memory and rows in lanes; at hd 512 they lie in
    // the shared part of Q, which is idle then
    static constexpr int STAGE = 32 * 128;
    static constexpr bool STAGE_IN_Q = HD == 512;
    // where three chunks of Q go to tensor memory the first group has a second one each, for its second chunk
    static constexpr int STAGES = HD == 256 && QT == 192 ? 12 : 8;
    static constexpr int BUF = NST * ENTRY + QS_BYTES + (STAGE_IN_Q ? 0 : STAGES * STAGE);
    static constexpr int O_COL = 0, S_COL = DV, P_COL = S_COL + 2 * kUnit, Q_COL = P_COL + PC * kUnit / 2;
    static_assert(Q_COL + QT / 2 <= 512, "tensor memory columns");
    // (the stages are the last two 64-element chunks of Q's shared part, which are written last)
    static_assert(!STAGE_IN_Q || (QS_BYTES >= 8 * STAGE && 8 * STAGE == 2 * kRowsP * 128), "the stages fit");
    // Everything else that is shared, behind the buffers: no static shared memory, so that the buffers begin where the
    // CTA's window does, at a multiple of 1024 (the kernel checks).
    struct Small {
        uint64_t bars[2 * NST + 14];
        unsigned long long odd[2];         // [group]: keys of its unit with a value that is not finite
        float base[2][kRowsP];             // [unit % 2][row]: the base after that unit
        float sum[2][kRowsP];              // [group][row]: the groups' sums at a piece's end
        int red[4][4];
        uint32_t tmem;
        int abort, acc;
    };
    static constexpr int SMEM = BUF + (int)sizeof(Small);
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

namespace {

__device__ __forceinline__ uint32_t ld_tmem_x1(uint32_t taddr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr) : "memory");
    return v;
}

// One lane of a converged warp.  The MMA warp runs as a whole and lets one lane issue: an MMA of 128 x 64 x 16 then
// takes 32 clocks to issue, against 46 where lane 0 alone runs the role (descriptors stay in uniform registers).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// or of a softmax group's flags, at its barrier
__device__ __forceinline__ bool any_of_group(bool v, int barrier) {
    int r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"((int)v), "r"(barrier) : "memory");
    return r != 0;
}
__device__ __forceinline__ void st_shared(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
// Both halves of a pair added to an f32, an instruction each.  (Converted first they cost 8 % of a causal prompt's time at
// hd 128; like this the sum of the rounded weights is as fast as that of the unrounded ones.)
__device__ __forceinline__ void add_pair(float& sum, uint32_t h2) {
    asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %1;\n\tadd.rn.f32.f16 %0, a, %0;\n\tadd.rn.f32.f16 %0, b, %0;\n\t}"
        : "+f"(sum) : "r"(h2));
}
// bit 15 of a half is set where the f16 value is not finite (its exponent field overflows by one)
__device__ __forceinline__ uint32_t not_finite(uint32_t v) { return (v & 0x7fff7fffu) + 0x04000400u; }

// The pieces of a CTA's stretch, walked alike by every role.
struct Walk {
    const Tile* tiles;
    long long left;
    int ntiles, head, ti, unit;   // head: KV head * CS + column part
    bool first;
    Tile t;
    int nu;                       // units of the piece: unit .. unit + nu - 1 of t

    __device__ __forceinline__ bool init(const Args& a) {
        const Hdr* h = hdr_of(a.plan);
        const Start& st = at<Start>(a.plan, a.d.start[1])[blockIdx.x];
        t = st.t;
        first = true;
        if (st.head < 0) return false;
        tiles = at<Tile>(a.plan, a.d.tiles[1]);
        ntiles = h->nt[1];
        head = st.head;
        ti = st.tile;
        unit = st.unit;
        left = min(h->u[1], h->wt[1] * a.d.nkv * a.d.cs - (long long)blockIdx.x * h->u[1]) - st.skip;
        return true;
    }
    __device__ __forceinline__ bool next() {
        while (left > 0) {
            if (ti == ntiles) {
                ti = 0;
                head++;
            }
            if (!first) t = tiles[ti];
            first = false;
            if (t.n > 0) break;
            ti++;
            unit = 0;
        }
        if (left <= 0) return false;
        nu = (int)min((long long)(t.n - unit), left);
        return true;
    }
    __device__ __forceinline__ void step() {
        left -= nu;
        unit += nu;
        if (unit == t.n) {
            left -= t.idle;
            unit = 0;
            ti++;
        }
    }
};

}  // namespace

template <int HD, bool PAIR>
__global__ void __launch_bounds__(kManyThreads, 1)
many_kernel(const Args a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using C = ManyCfg<HD, PAIR>;
    extern __shared__ __align__(1024) uint8_t smem[];
    auto& sm = *reinterpret_cast<typename C::Small*>(smem + C::BUF);
    const Dims& d = a.d;
    const Hdr* h = hdr_of(a.plan);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // The next kernel may begin: it reads nothing of this one, and waits for its end before it ends itself.
    pdl_launch_dependents();
    if (!plan_fits(h, d)) {
        if (blockIdx.x == 0 && tid == 0) atomicOr(&g_status_paged_mma, kStatusPlan);
        return;
    }
    Walk w;
    if (!w.init(a)) return;
    const uint32_t ring = smem_u32(smem);
    if (ring & 1023u) {                      // the swizzled tiles need it; never the case
        if (tid == 0) atomicOr(&g_status_paged_mma, kStatusTimeout);
        return;
    }
    const uint32_t qs = ring + C::NST * C::ENTRY;                    // the part of Q that is not in tensor memory
    const uint32_t stages = qs + (C::STAGE_IN_Q ? C::QS_BYTES - 8 * C::STAGE : C::QS_BYTES);
    const uint32_t bar0 = smem_u32(sm.bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (C::NST + s); };
    const uint32_t b_s = bar0 + 8u * (2 * C::NST);                   // [2] scores of a unit are there
    const uint32_t b_read = b_s + 16;                                // [2] and have been read
    const uint32_t b_base = b_s + 32;                                // [2] the rows' bases are set
    const uint32_t b_pv = b_s + 48;                                  // [2] the unit's product is added
    const uint32_t b_p = b_s + 64;                                   // its weights are there
    const uint32_t b_q = b_s + 72;                                   // the piece's Q is there
    const uint32_t b_o = b_s + 80;                                   // the piece's products are all added
    const uint32_t b_drain = b_s + 88;                               // [2] winding down
    // The piece's result has been read out of O.  Each group reads half of the columns, for as long as its stores take, and
    // the group that has the next piece's first unit goes on alone: its weights (b_p) say nothing of the other group's
    // reading.  So a piece's first product, which overwrites all of O, waits here for the eight warps; later ones, and the
    // rescaling before them, come behind that product.
    const uint32_t b_out = b_s + 104;
    if (tid == 0) {
        for (int i = 0; i < 2 * C::NST; i++) mbar_init(bar0 + 8u * i, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(b_s + 8 * i, 1);
            mbar_init(b_read + 8 * i, kGroup / 32);
            mbar_init(b_base + 8 * i, kGroup / 32);
            mbar_init(b_pv + 8 * i, 1);
        }
        mbar_init(b_p, kGroup / 32);
        mbar_init(b_q, kSoft / 32);
        mbar_init(b_o, 1);
        mbar_init(b_drain, 1);
        mbar_init(b_drain + 8, 1);
        mbar_init(b_out, kSoft / 32);
        fence_mbar_init();
        sm.abort = 0;
    }
    if (warp == 9) {
        tc::tmem_alloc(smem_u32(&sm.tmem), 512);
        tc::tmem_relinquish();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* abort = &sm.abort;
    unsigned* status = &g_status_paged_mma;
    const int pl = h->prefix_len, G = d.G;

    if (warp == 8 || warp == 11) {
        // ---------------------------------------------------------------- TMA: warp 8 K, warp 11 V
        // (One warp for both took 1.3 us a unit, most of it issue and lookup latency: longer than the unit's MMAs.)
        const bool is_v = warp == 11;
        const int first = is_v ? C::NK : 0, slots = is_v ? C::NV : C::NK, entries = is_v ? C::VE : C::KE;
        const CUtensorMap* map = is_v ? &vmap : &kmap;
        int slot = 0, used = 0;                   // the ring's next slot; slots that were ever filled
        uint32_t turn = 0;                        // parity of the ring's round
        bool ok = true;
        // A page gives `box` rows of a unit at a time.  One copy brings all of an entry's columns of a V box, and of a
        // whole K unit; where a unit has several boxes K takes a copy per 64-column chunk as well, so that a chunk's
        // 64 rows lie together.  Each lane has one copy.
        const int box = min(d.ps, kUnit), boxes = kUnit / box, lboxes = __ffs(boxes) - 1;
        const int my_p = lane & (boxes - 1), my_c = is_v ? 0 : lane >> lboxes;
        const bool issues = is_v || boxes == 1 ? lane < boxes : my_c < C::EC / 64;
        const uint32_t my_dst = ring + first * C::ENTRY + (is_v ? my_p * box * (C::EC * 2) : my_c * (kUnit * 128) + my_p * box * 128);
        while (ok && w.next()) {
            const int head = w.head / C::CS, chunk0 = (is_v ? w.head % C::CS * C::DV / 64 : 0) + my_c;
            int ids = -1, ids_at = -64;           // 32 page ids from ids_at on, a lane each
            bool ids_pre = false;
            #pragma unroll 1
            for (int u = 0; u < w.nu && ok; u++) {
                const Unit un = unit_of(w.t, w.unit + u);
                const int page0 = un.key >> d.lps, last = (un.key + kUnit - 1) >> d.lps;
                if (un.pre != ids_pre || last >= ids_at + 32) {
                    const int* table = un.pre ? a.pre_table : a.table + (size_t)w.t.seq * d.own_pages;
                    ids_pre = un.pre;
                    ids_at = page0;
                    ids = ids_at + lane < (un.pre ? d.pre_pages : d.own_pages) ? __ldg(table + ids_at + lane) : -1;
                }
                const int k = un.key + my_p * box;
                const int id = __shfl_sync(0xffffffffu, ids, (k >> d.lps) - ids_at);
                const int at_row = cache_row(id, a.num_pages, d.nkv, d.lps, head, k);
                const int row = at_row < 0 ? a.num_pages * d.nkv * d.ps : at_row;   // past the map: zeros
                #pragma unroll 1
                for (int e = 0; e < entries; e++) {
                    // from the second round on: the slot's MMAs of the round before are done
                    if (used == slots)
                        ok = wait_warp(empty(first + slot), turn ^ 1u, abort, status);
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(full(first + slot), C::ENTRY);
                    __syncwarp();
                    if (issues)
                        tma_chunks(my_dst + slot * C::ENTRY, map, row, chunk0 + e * (C::EC / 64), full(first + slot));
                    used = max(used, slot + 1);
                    if (++slot == slots) {
                        slot = 0;
                        turn ^= 1u;
                    }
                }
            }
            w.step();
        }
        __syncwarp();
        // every copy lands before the CTA gives up its shared memory
        for (int s = 0; s < used; s++)            // the slots before the next one were filled in this round
            mbar_wait_drain(full(first + s), s < slot ? turn : turn ^ 1u, status);
    } else if (warp == 9 || warp == 10) {
        // ---------------------------------------------------------------- MMA: warp 9 the scores, warp 10 the products
        // Two warps, because one's waits would leave the tensor core without work: a unit's 1,100 clocks of MMAs took
        // 2,300 with one.
        const bool products = warp == 10;
        constexpr uint32_t id_s = tc::idesc(1, 0, 0, 0, 0, kUnit, kRowsP);
        constexpr uint32_t id_o = tc::idesc(1, 0, 0, 0, 1, C::EC, kRowsP);
        int slot = 0;                              // the next entry's
        uint32_t turn = 0;                         // parity of the ring's round
        uint32_t it = 0, piece = 0;                // units and pieces so far
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = ok && wait_warp(bar, parity, abort, status);
            tc::fence_after();
        };
        auto entry = [&]() {                       // the next entry of this warp's ring, once it has landed
            const int s = (products ? C::NK : 0) + slot;
            wait(full(s), turn);
            if (++slot == (products ? C::NV : C::NK)) {
                slot = 0;
                turn ^= 1u;
            }
            return s;
        };
        // A descriptor's address field counts 16 bytes and has room for all of shared memory: the descriptors of an
        // entry's tiles are its first one's plus a constant.
        // V lies box by box: chunks of `box` rows, 16 keys (two groups of 8 rows of 128 bytes) at a time.
        const int box = min(d.ps, kUnit);
        const uint64_t k_desc = tc::sdesc_sw128(ring, 16, 1024), v_desc = tc::sdesc_sw128(ring, box * 128, 1024);
        uint32_t v_off[kUnit / 16];
        #pragma unroll
        for (int k = 0; k < kUnit / 16; k++)
            v_off[k] = (uint32_t)((16 * k) / box * box * (C::EC * 2) + (16 * k) % box * 128) / 16;
        const uint64_t q_desc = tc::sdesc_sw128(qs, 16, 1024);
        auto scores = [&](uint32_t i) {            // i: units before this one, all pieces'
            if (i >= 2) wait(b_read + 8u * (i & 1u), ((i >> 1) - 1) & 1u);     // its buffer's last scores have been read
            const uint32_t ds = tmem + C::S_COL + (i & 1u) * kUnit;
            #pragma unroll
            for (int pe = 0; pe < C::KE; pe++) {
                const int s = entry();
                if (!ok) return;
                const uint64_t kd = k_desc + (uint64_t)(s * (C::ENTRY / 16));
                if (elect_one()) {
                    #pragma unroll
                    for (int k = 0; k < C::EC / 16; k++) {
                        const int e = pe * C::EC + 16 * k;                     // element of the head
                        const uint64_t bd = kd + (uint64_t)((k / 4) * (kUnit * 128 / 16) + (k % 4) * 2);
                        if (e < C::QT)
                            tc::mma_f16_ts(ds, tmem + C::Q_COL + e / 2, bd, id_s, e > 0);
                        else
                            tc::mma_f16_ss(ds, q_desc + (uint64_t)(((e - C::QT) / 64) * (kRowsP * 128 / 16) + (k % 4) * 2), bd,
                                           id_s, 1);
                    }
                    tc::commit(empty(s));
                    if (pe == C::KE - 1) tc::commit(b_s + 8u * (i & 1u));
                }
                __syncwarp();
            }
        };
        auto product = [&](int u) {
            int acc = 1;
            if (u == 0 && piece > 1) wait(b_out, piece & 1u);      // (piece counts this one: the last but one's phase)
            #pragma unroll
            for (int ve = 0; ve < C::VE; ve++) {
                const int s = entry();             // (V is there long before the weights: that wait comes first)
                if (ve == 0) {
                    wait(b_p, (it + u) & 1u);
                    if (u == 0) acc = *(volatile int*)&sm.acc;
                }
                if (!ok) return;
                const uint64_t vd = v_desc + (uint64_t)(s * (C::ENTRY / 16));
                if (elect_one()) {
                    #pragma unroll
                    for (int p = 0; p < C::PC; p++)            // the weights' high parts, the low ones
                        #pragma unroll
                        for (int k = 0; k < kUnit / 16; k++)
                            tc::mma_f16_ts(tmem + C::O_COL + ve * C::EC, tmem + C::P_COL + p * (kUnit / 2) + 8 * k, vd + v_off[k],
                                           id_o, acc || p + k > 0);
                    if (ve == C::VE - 1) tc::commit(b_pv + 8u * ((it + u) & 1u));
                    tc::commit(empty(s));
                    if (ve == C::VE - 1 && u == w.nu - 1) tc::commit(b_o);
                }
                __syncwarp();
            }
        };
        while (ok && w.next()) {
            if (!products) wait(b_q, piece & 1u);
            piece++;
            #pragma unroll 1
            for (int u = 0; ok && u < w.nu; u++) {
                if (products) product(u);
                else scores(it + u);               // up to two units ahead: a buffer is free as soon as it has been read
            }
            it += w.nu;
            w.step();
        }
        // every MMA is done before the CTA gives up its tensor memory
        if (elect_one()) tc::commit(b_drain + 8u * products);
        __syncwarp();
        mbar_wait_drain(b_drain + 8u * products, 0, status);
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- softmax: two groups
        // A unit is one group's, a thread per row; the groups take units in turn, so that one's loads, exchanges and
        // stores run beside the other's exponentials.  A row's base passes from group to group with each unit.  (Q and the
        // result are halved by columns instead.)
        const int half = warp >> 2, wq = warp & 3, r0 = wq * 32 + lane;
        const uint32_t tl = tmem + ((uint32_t)(wq * 32) << 16);      // this warp's lanes
        constexpr int DH = C::DV / 2;                                // columns of the result that this warp writes
        const int group_bar = 2 + half;                              // the group's named barrier; 1 is both's
        auto group_sync = [&]() { named_bar_sync(2 + half, kGroup); };
        // one arrival per warp: 32 lanes' on one barrier would come one after the other
        auto arrive = [&](uint32_t bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        const uint32_t stage = stages + (C::STAGES == 12 && half == 0 ? 2 * warp : C::STAGES - 8 + warp) * C::STAGE;
        uint32_t it = 0, pieces = 0;              // units and pieces so far
        // A wait that ran out clears ok.  The warp then walks on without waiting, so that the warps meet at
        // the same named barriers to the end; it writes no result.
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = ok && wait_warp(bar, parity, abort, status);
        };
        // The product of a unit is added, waited for by the next unit's group.  (A parity tells a barrier's phase from the
        // one before only: with a barrier for each group's units, none is skipped.)
        auto wait_pv = [&](uint32_t unit) {
            wait(b_pv + 8u * (unit & 1u), (unit >> 1) & 1u);
            tc::fence_after();
        };
        // Q of the piece that w stands at: its rows into tensor memory (two elements per column) and, past QT, shared
        // memory.  All that has a place at once is on its way at once (a chunk after the other took 1,650 clocks each).
        // Eight lanes read 128 bytes of a row; a stage turns rows over lanes into a row per lane.
        unsigned alive = 0;      // this warp's rows that the piece is for: a prefix tile may span rows that are not
        auto load_q = [&](int row) {
            const long long mine = ((long long)(row / G) * a.q_stride + (long long)((w.head / C::CS) * G + row % G) * HD) * 2;
            const char* qb = reinterpret_cast<const char*>(a.q) + (lane & 7) * 16;
            auto fetch = [&](int c, uint32_t to) {             // chunk c: 64 elements
                #pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int r = 4 * i + (lane >> 3);         // of the warp's rows
                    const char* src = qb + __shfl_sync(0xffffffffu, mine, r) + c * 128;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + r * 128 + (((lane & 7) ^ (r & 7)) << 4)),
                                 "l"(src), "r"((alive >> r) & 1u ? 16 : 0)      // 0: zeros
                                 : "memory");
                }
            };
            auto landed = [&]() {
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
            };
            auto to_tmem = [&](int c, uint32_t from) {
                uint32_t v[32];
                #pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint4 y = ld_shared(from + lane * 128 + ((j ^ (lane & 7)) << 4));
                    v[4 * j] = y.x;
                    v[4 * j + 1] = y.y;
                    v[4 * j + 2] = y.z;
                    v[4 * j + 3] = y.w;
                }
                tc::st_32x32b_x32(tl + C::Q_COL + 32 * c, v);
                __syncwarp();
            };
            constexpr int QC = C::QT / 64;                     // chunks in tensor memory
            auto shared_of = [&](int c) { return qs + (c - QC) * (kRowsP * 128) + wq * (32 * 128); };
            constexpr int NC = HD / 128;                       // chunks of this half
            // (loops that stay loops: code that runs once comes from memory as slowly as data does)
            if constexpr (!C::STAGE_IN_Q) {
                #pragma unroll 1
                for (int n = 0; n < NC; n++) {
                    const int c = half + 2 * n;
                    fetch(c, c < QC ? stage + n * C::STAGE : shared_of(c));
                }
                landed();
                #pragma unroll 1
                for (int n = 0; n < NC && half + 2 * n < QC; n++) to_tmem(half + 2 * n, stage + n * C::STAGE);
            } else {
                // chunks by turns; the last one of each half goes where the stages are, when those are done with
                #pragma unroll 1
                for (int n = 0; n < NC; n++) {
                    const int c = half + 2 * n;
                    if (n == NC - 1) named_bar_sync(1, kSoft);
                    fetch(c, c < QC ? stage : shared_of(c));
                    if (c < QC) {
                        landed();
                        to_tmem(c, stage);
                    }
                }
                landed();
            }
            if constexpr (HD > C::QT) tc::fence_proxy_async_smem();
            tc::wait_st();
            tc::fence_before();
            arrive(b_q);
        };
        // A piece's result is written after the next piece's Q has been loaded (its scores are made meanwhile), except
        // at hd 512, where the stages lie in Q's place.
        bool more = w.next(), pending = false;
        float m = -INFINITY, l = 0.f;
        unsigned mask = 0;                        // the pending result's rows,
        char* dst = nullptr;                      // where they go,
        size_t mine = 0;                          // this row's offset there,
        float2* ml = nullptr;                     // its (base, sum), null where the result is finished here,
        int esize = 4;                            // the bytes of an element
        for (;;) {
            // What the next piece needs from memory is asked for before the result of the last one is written.
            const int part = w.head % C::CS, nrows = w.t.nrows, row = w.t.row0 + min(r0, nrows - 1);
            const int tok = row / G, hq = (w.head / C::CS) * G + row % G;
            const int u0 = (int)((it ^ (uint32_t)half) & 1u);        // this group's first unit
            // page ids of a unit, one per box, in the first lanes; fetched a unit ahead
            const int box = min(d.ps, kUnit), boxes = kUnit / box;
            auto page_of = [&](int u) {
                if (u >= w.nu) return -1;
                const Unit un = unit_of(w.t, w.unit + u);
                const int idx = (un.key + (lane & 3) * box) >> d.lps;
                const int* table = un.pre ? a.pre_table : a.table + (size_t)w.t.seq * d.own_pages;
                return lane < boxes && idx < (un.pre ? d.pre_pages : d.own_pages) ? __ldg(table + idx) : -1;
            };
            int page = -1, vlo = 0, vhi = 0;          // the positions that this row sees, [vlo, vhi)
            if (more) {
                const int pos = __ldg(at<int>(a.plan, d.tok_pos) + tok);
                const int pre = w.t.seq >= 0 ? 0 : __ldg(at<int>(a.plan, d.row_pre) + row);
                page = page_of(u0);
                const bool live = r0 < nrows && pre != -1;
                alive = __ballot_sync(0xffffffffu, live);
                vhi = live ? pos + 1 : 0;
                vlo = live && d.window > 0 ? max(0, pos + 1 - d.window) : 0;
            }
            // the last unit's scores, which may be the other group's, are made: Q may be written over
            if (pending) wait(b_s + 8u * ((it - 1) & 1u), ((it - 1) >> 1) & 1u);
            if (!C::STAGE_IN_Q && more) load_q(row);
            // Both groups' sums, on the last unit's base.  Behind this wait every warp has taken up the last piece, and has
            // read what is shared about it: a piece of one unit, which one group does alone, has a barrier for that.
            if (pending) {
                wait(b_base + 8u * ((it - 1) & 1u), ((it - 1) >> 1) & 1u);
                const float last = sm.base[(it - 1) & 1][r0];
                if (m != last && l != 0.f) l *= exp2_approx(m - last);
                m = last;
                sm.sum[half][r0] = l;
            }
            if (more && half == 0) {
                const bool live = (alive >> lane) & 1u;
                // what all rows see, what any row sees
                const int4 seen = make_int4(__reduce_max_sync(0xffffffffu, vlo), __reduce_min_sync(0xffffffffu, live ? vhi : 0x7fffffff),
                                            __reduce_min_sync(0xffffffffu, live ? vlo : 0x7fffffff), __reduce_max_sync(0xffffffffu, vhi));
                if (lane == 0) {
                    sm.red[wq][0] = seen.x;
                    sm.red[wq][1] = seen.y;
                    sm.red[wq][2] = seen.z;
                    sm.red[wq][3] = seen.w;
                }
            }
            named_bar_sync(1, kSoft);
            if (pending) {
                l = sm.sum[0][r0] + sm.sum[1][r0];
                wait(b_o, (pieces - 1) & 1u);
                tc::fence_after();
                const float inv = ml ? 1.f : l == 0.f ? 0.f : 1.f / l;
                if (((mask >> lane) & 1u) && ok && ml && half == 0) *ml = make_float2(m, l);
                // 128 bytes of every row of the warp, from a row per lane to eight lanes per row
                const int per = 128 / esize;      // columns
                #pragma unroll 1
                for (int c = half * DH; c < (half + 1) * DH; c += per) {
                    uint32_t v[32];
                    tc::ld_32x32b_x32(tl + C::O_COL + c, v);
                    tc::wait_ld();
                    #pragma unroll
                    for (int j = 0; j < 32; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) * inv);
                    if (esize == 2) {
                        uint32_t y[32];
                        tc::ld_32x32b_x32(tl + C::O_COL + c + 32, y);
                        tc::wait_ld();
                        #pragma unroll
                        for (int j = 0; j < 16; j++) {
                            v[j] = half_pair(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                            y[j] = half_pair(__uint_as_float(y[2 * j]) * inv, __uint_as_float(y[2 * j + 1]) * inv);
                        }
                        #pragma unroll
                        for (int j = 0; j < 16; j++) v[16 + j] = y[j];
                    }
                    if (c + per == (half + 1) * DH) {
                        tc::fence_before();           // this warp has read O, for the product that overwrites it
                        arrive(b_out);
                    }
                    #pragma unroll
                    for (int j = 0; j < 8; j++)
                        st_shared(stage + lane * 128 + ((j ^ (lane & 7)) << 4),
                                  make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
                    __syncwarp();
                    #pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int r = 4 * i + (lane >> 3);
                        const uint4 x = ld_shared(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                        const size_t o = __shfl_sync(0xffffffffu, mine, r) + (size_t)c * esize;
                        if (ok && (mask >> r) & 1u) *reinterpret_cast<uint4*>(dst + o + (lane & 7) * 16) = x;
                    }
                    __syncwarp();
                }
                tc::fence_before();
                if (C::STAGE_IN_Q) named_bar_sync(1, kSoft);   // every stage has been emptied
            }
            if (C::STAGE_IN_Q && more) load_q(row);
            if (!more) break;
            mask = alive;
            int all_lo = 0, all_hi = 0x7fffffff, any_lo = 0x7fffffff, any_hi = 0;
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                all_lo = max(all_lo, sm.red[i][0]);
                all_hi = min(all_hi, sm.red[i][1]);
                any_lo = min(any_lo, sm.red[i][2]);
                any_hi = max(any_hi, sm.red[i][3]);
            }
            if (w.nu == 1) named_bar_sync(1, kSoft);
            m = -INFINITY;
            l = 0.f;
            const uint32_t it0 = it;
            #pragma unroll 1
            for (int u = u0; u < w.nu; u += 2) {
                it = it0 + u;
                const Unit un = unit_of(w.t, w.unit + u);
                const int key = un.pre ? un.key : un.key + pl, end = un.pre ? un.hi : un.hi + pl;   // as positions
                const unsigned there = __ballot_sync(0xffffffffu, lane < boxes && page >= 0 && page < a.num_pages);
                page = page_of(u + 2);
                const bool edge = there != (1u << boxes) - 1 || key < all_lo || key + kUnit > min(all_hi, end);
                wait(b_s + 8u * half, (it >> 1) & 1u);
                tc::fence_after();
                const uint32_t ts = tl + C::S_COL + half * kUnit;
                uint32_t x[2][32];
                tc::ld_32x32b_x32(ts, x[0]);
                tc::ld_32x32b_x32(ts + 32, x[1]);
                tc::wait_ld();
                tc::fence_before();
                arrive(b_read + 8u * half);
                if (edge) {
                    // the keys that this row sees, one bit each
                    auto below = [&](int k) { return k >= kUnit ? ~0ull : k <= 0 ? 0ull : (1ull << k) - 1; };
                    unsigned long long bits = below(min(vhi, end) - key) & ~below(vlo - key);
                    if (there != (1u << boxes) - 1)
                        for (int b = 0; b < boxes; b++)
                            if (!((there >> b) & 1u)) bits &= ~(below((b + 1) * box) & ~below(b * box));
                    #pragma unroll
                    for (int k = 0; k < 2; k++)
                        #pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (!(((uint32_t)(bits >> (32 * k)) >> j) & 1u)) x[k][j] = 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                #pragma unroll
                for (int j = 0; j < 32; j++) {
                    mx[j & 1] = fmaxf(mx[j & 1], __uint_as_float(x[0][j]));
                    mx[2 + (j & 1)] = fmaxf(mx[2 + (j & 1)], __uint_as_float(x[1][j]));
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale;
                // The base that the other group left, or a new one.  Units so far of this piece are in O: rescale it where
                // a row's maximum has left its base behind.  A row that saw nothing yet has zeros there and in l.
                if (it > 0) wait(b_base + 8u * (half ^ 1), ((it - 1) >> 1) & 1u);
                const float from = u > 0 ? sm.base[half ^ 1][r0] : -INFINITY;
                if (m != from && l != 0.f) l *= exp2_approx(m - from);
                // A warp that has a row to rescale takes the base after every row's maximum that has grown: it is the warp
                // that pays, and this way seldom twice.
                // (differences: a sum of the base and 15 may round up past the largest weight)
                const bool any = __any_sync(0xffffffffu, top - from > kMost && from != -INFINITY);
                const bool set = u == 0 || from == -INFINITY || (any && top - from > kLift), scale = set && from != -INFINITY;
                m = set ? top - kLift : from;
                sm.base[half][r0] = m;
                arrive(b_base + 8u * half);
                const float base0 = m == -INFINITY ? 0.f : m;
                const bool far = fabsf(base0) >= kFar;
                if (__any_sync(0xffffffffu, far)) {
                    #pragma unroll
                    for (int k = 0; k < 2; k++)
                        #pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (far) x[k][j] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(x[k][j]), a.scale), base0));
                }
                const float slope = far ? 1.f : a.scale, base = far ? 0.f : base0;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t low[32];
                #pragma unroll
                for (int k = 0; k < 2; k++)
                    #pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const float e0x = exp2_approx(fmaf(__uint_as_float(x[k][2 * j]), slope, -base));
                        const float e1x = exp2_approx(fmaf(__uint_as_float(x[k][2 * j + 1]), slope, -base));
                        const uint32_t h2 = half_pair(e0x, e1x);
                        x[0][16 * k + j] = h2;                        // P over the scores it is made of
                        if constexpr (PAIR) {
                            sum[j & 3] += e0x + e1x;
                            low[16 * k + j] = half_pair(e0x - h_lo(h2), e1x - h_hi(h2));
                        } else {
                            add_pair(sum[j & 3], h2);
                        }
                    }
                if (scale) l *= exp2_approx(from - m);
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                // The unit before is in O, and its P may be written over.  (Behind a piece's first unit it is the piece before's:
                // done, but its phase is counted.)
                if (it > 0) wait_pv(it - 1);
                tc::st_32x32b_x32(tl + C::P_COL, x[0]);
                if constexpr (PAIR) tc::st_32x32b_x32(tl + C::P_COL + kUnit / 2, low);
                if (any) {
                    // the next 32 columns come while these are stored
                    const float f = scale ? exp2_approx(from - m) : 1.f;
                    uint32_t o[2][32];
                    tc::ld_32x32b_x32(tl + C::O_COL, o[0]);
                    #pragma unroll 1
                    for (int c = 0; c < C::DV; c += 64) {
                        #pragma unroll
                        for (int k = 0; k < 2; k++) {
                            tc::wait_ld();
                            if (k == 0 || c + 64 < C::DV) tc::ld_32x32b_x32(tl + C::O_COL + c + 32 * (k + 1), o[k ^ 1]);
                            #pragma unroll
                            for (int j = 0; j < 32; j++) o[k][j] = __float_as_uint(__uint_as_float(o[k][j]) * f);
                            tc::st_32x32b_x32(tl + C::O_COL + c + 32 * k, o[k]);
                        }
                    }
                }
                if (u == 0 && r0 == 0) *(volatile int*)&sm.acc = 0;
                if (edge) {
                    // Values that no row sees become zeros; values that only some rows see and that are not
                    // finite (0 x NaN is not 0) are added row by row here and then cleared.
                    // (V of the unit before has landed, or its product were not done: the parity is this phase's.)
                    uint32_t v_at[C::VE];
                    #pragma unroll
                    for (int ve = 0; ve < C::VE; ve++) {
                        const uint32_t n = it * C::VE + ve, s = C::NK + n % C::NV;
                        wait(full(s), (n / C::NV) & 1u);
                        v_at[ve] = ring + s * C::ENTRY;
                    }
                    // this thread's share: 16 bytes (r0 % 8) of keys r0 / 8 + 16 r in each 64-column chunk
                    auto key_at = [&](int c, int k) {        // key k's 128 bytes of chunk c
                        return v_at[c / (C::EC / 64)] + (k & ~(box - 1)) * (C::EC * 2) + c % (C::EC / 64) * box * 128 +
                               (k & (box - 1)) * 128;
                    };
                    auto piece_at = [&](int c, int r) { return key_at(c, (r0 >> 3) + 16 * r) + (r0 & 7) * 16; };
                    uint32_t bad = 0;
                    bool some[4], none[4], clear = false;    // key r is seen by some rows only, by none
                    #pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int k = key + (r0 >> 3) + 16 * r;
                        none[r] = k < any_lo || k >= min(any_hi, end);
                        some[r] = !none[r] && (k < all_lo || k >= all_hi);
                        clear |= none[r];
                    }
                    #pragma unroll
                    for (int c = 0; c < C::DV / 64; c += 2) {
                        uint4 v[8];                          // eight loads under way, needed or not
                        #pragma unroll
                        for (int i = 0; i < 8; i++) v[i] = ld_shared(piece_at(c + (i >> 2), i & 3));
                        #pragma unroll
                        for (int i = 0; i < 8; i++)
                            if (some[i & 3]) bad |= not_finite(v[i].x) | not_finite(v[i].y) | not_finite(v[i].z) | not_finite(v[i].w);
                    }
                    if (clear) {
                        #pragma unroll
                        for (int r = 0; r < 4; r++)
                            for (int c = 0; c < C::DV / 64 && none[r]; c++) st_shared(piece_at(c, r), make_uint4(0, 0, 0, 0));
                    }
                    unsigned long long odd = 0;
                    if (any_of_group((bad & 0x80008000u) != 0, group_bar)) {
                        if (r0 == 0) sm.odd[half] = 0;
                        group_sync();
                        for (int r = 0; r < 4; r++)
                            for (int c = 0; c < C::DV / 64 && some[r]; c++) {
                                const uint4 v = ld_shared(piece_at(c, r));
                                if ((not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w)) & 0x80008000u)
                                    atomicOr(&sm.odd[half], 1ull << ((r0 >> 3) + 16 * r));
                            }
                        group_sync();
                        odd = *(volatile unsigned long long*)&sm.odd[half];
                    }
                    if (odd) {
                        tc::wait_st();                       // P, read back below
                        if (u == 0) {
                            if (pieces > 0) {                // the other group's columns too are overwritten
                                wait(b_out, (pieces - 1) & 1u);
                                tc::fence_after();
                            }
                            uint32_t z[32];
                            #pragma unroll
                            for (int j = 0; j < 32; j++) z[j] = 0;
                            #pragma unroll 1
                            for (int c = 0; c < C::DV; c += 32) tc::st_32x32b_x32(tl + C::O_COL + c, z);
                            tc::wait_st();
                            if (r0 == 0) *(volatile int*)&sm.acc = 1;
                        }
                        for (unsigned long long rest = odd; rest; rest &= rest - 1) {
                            const int j = __ffsll((long long)rest) - 1;
                            float pf = 0.f;
                            #pragma unroll
                            for (int p = 0; p < C::PC; p++) {
                                const uint32_t pj = ld_tmem_x1(tl + C::P_COL + p * (kUnit / 2) + j / 2);
                                tc::wait_ld();
                                pf += j & 1 ? h_hi(pj) : h_lo(pj);
                            }
                            const bool sees = key + j >= vlo && key + j < min(vhi, end) && ((there >> (j / box)) & 1u);
                            #pragma unroll 1
                            for (int c = 0; c < C::DV; c += 32) {
                                uint32_t o[32];
                                tc::ld_32x32b_x32(tl + C::O_COL + c, o);
                                tc::wait_ld();
                                const uint32_t vr = key_at(c / 64, j);
                                #pragma unroll
                                for (int q = 0; q < 4; q++) {
                                    const int un = (c % 64) / 8 + q;
                                    const uint4 v = ld_shared(vr + ((un ^ (j & 7)) << 4));
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
                        group_sync();                        // every row has read the values
                        for (int r = 0; r < 4; r++)
                            for (int c = 0; c < C::DV / 64; c++)
                                if ((odd >> ((r0 >> 3) + 16 * r)) & 1ull)
                                    st_shared(piece_at(c, r), make_uint4(0, 0, 0, 0));
                    }
                    if (odd || key < any_lo || key + kUnit > min(any_hi, end)) tc::fence_proxy_async_smem();   // V was written
                }
                tc::wait_st();
                tc::fence_before();
                arrive(b_p);
            }
            it = it0 + w.nu;
            pieces++;
            // where the row's result goes: finished, or this stretch's part of it
            const bool whole = w.nu == w.t.n, direct = whole && w.t.solo;
            const size_t at_slot = whole ? ((size_t)(w.t.seq < 0 ? 0 : 1) * d.T + tok) * d.nH + hq
                                         : ((size_t)blockIdx.x * 2 + (w.unit == 0 ? 1 : 0)) * kRowsP + r0;
            dst = reinterpret_cast<char*>(!direct ? whole ? a.w.row : a.w.edge[1] : a.out);
            ml = direct ? nullptr : whole ? a.w.row_ml + at_slot * 2 + part : a.w.edge_ml[1] + at_slot;
            esize = direct && !a.out_f32 ? 2 : 4;
            mine = (size_t)esize * (!direct ? whole ? at_slot * HD + part * C::DV : at_slot * C::DV
                                            : (size_t)tok * a.out_stride + (size_t)hq * HD + part * C::DV);
            pending = true;
            w.step();
            more = w.next();
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 9) tc::tmem_dealloc(tmem, 512);
}

template <int HD>
static cudaError_t launch(const Args& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
    const auto kernel = a.out_f32 ? many_kernel<HD, true> : many_kernel<HD, false>;
    const int smem = a.out_f32 ? ManyCfg<HD, true>::SMEM : ManyCfg<HD, false>::SMEM;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    kernel<<<a.d.ctas[1], kManyThreads, smem, s>>>(a, km, vm);
    return cudaGetLastError();
}

int launch_many(const Args& a, cudaStream_t s) {
    CUtensorMap km, vm;
    const uint64_t rows = (uint64_t)a.num_pages * a.d.nkv * a.d.ps;
    for (int i = 0; i < 2; i++) {
        const int box = a.d.ps < kUnit ? a.d.ps : kUnit, chunks = (a.d.hd == 256 ? 256 : 128) / 64;   // of an entry
        const int st = tensor_map_chunks(i ? &vm : &km, i ? a.vc : a.kc, a.d.hd, rows, box, i || box == kUnit ? chunks : 1);
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
