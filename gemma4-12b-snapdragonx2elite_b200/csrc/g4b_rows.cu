// g4b_rows.cu -- the prefill layer's element-wise dispatches over [M, D] rows of tokens:
//   rows_rmsnorm   vk/pre_norm.comp:8-13    y[m] = x[m] * rsqrt(mean(x[m]^2) + 1e-6) * w
//   rows_normadd   vk/pre_na.comp:9-15      h[m] = (h[m] + x[m] * rsqrt(mean(x[m]^2) + 1e-6) * w) * scl
//   gelumul        vk/gelumul.comp:7-8      out = gelu_tanh(gate) * up, element-wise
//   rows_normadd_i8  rows_normadd, the next rows_rmsnorm and cast_i8 (vk/cast_i8.comp:11-19) in one pass
// recorded around each layer's prefill GEMMs (src/vk_engine.py:413-424).
//
// All three are HBM-bound streams.  The two norms run one CTA per row: a vectorised sum-of-squares
// pass, a block reduction, then a second pass over the same row (L1/L2-resident by then), so HBM sees
// each byte once.  x and y / out may be f32 or f16 (the GEMMs' operands); the residual h is f32, as in
// the engine.
#include <algorithm>

#include "g4b_common.cuh"

namespace g4b {

constexpr int kRowThreads = 256;
constexpr float kRowEps = 1e-6f;   // vk/pre_norm.comp:12, vk/pre_na.comp:13

// 4 consecutive values as f32 / stored from f32
template <bool F32>
__device__ __forceinline__ float4 ld4(const void* p, size_t i4) {
    if constexpr (F32) return __ldg(reinterpret_cast<const float4*>(p) + i4);
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p) + i4);
    return make_float4(h_lo(u.x), h_hi(u.x), h_lo(u.y), h_hi(u.y));
}
template <bool F32>
__device__ __forceinline__ void st4(void* p, size_t i4, float4 v) {
    if constexpr (F32) {
        reinterpret_cast<float4*>(p)[i4] = v;
    } else {
        uint2 u;
        u.x = pack_half2(__float2half_rn(v.x), __float2half_rn(v.y));
        u.y = pack_half2(__float2half_rn(v.z), __float2half_rn(v.w));
        reinterpret_cast<uint2*>(p)[i4] = u;
    }
}

// rsqrt(mean(x^2) + eps) of the CTA's row (x as f32 or f16, D % 4 == 0)
template <bool XF32>
__device__ __forceinline__ float row_inv_rms(const void* x, size_t row4, int D4, float* red) {
    float s = 0.f;
    for (int i = threadIdx.x; i < D4; i += kRowThreads) {
        const float4 v = ld4<XF32>(x, row4 + i);
        s = fmaf(v.x, v.x, s);
        s = fmaf(v.y, v.y, s);
        s = fmaf(v.z, v.z, s);
        s = fmaf(v.w, v.w, s);
    }
    #pragma unroll
    for (int m = 16; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    float tot = 0.f;
    #pragma unroll
    for (int w = 0; w < kRowThreads / 32; w++) tot += red[w];
    return rsqrtf(tot / (float)(4 * D4) + kRowEps);
}

template <bool XF32, bool YF32>
__global__ void __launch_bounds__(kRowThreads) rows_rmsnorm_kernel(const void* __restrict__ x,
                                                                  const float* __restrict__ w, void* __restrict__ y,
                                                                  int D) {
    __shared__ float red[kRowThreads / 32];
    const int D4 = D / 4;
    const size_t row4 = (size_t)blockIdx.x * D4;
    const float inv = row_inv_rms<XF32>(x, row4, D4, red);
    for (int i = threadIdx.x; i < D4; i += kRowThreads) {
        const float4 v = ld4<XF32>(x, row4 + i), g = __ldg(reinterpret_cast<const float4*>(w) + i);
        st4<YF32>(y, row4 + i, make_float4(v.x * inv * g.x, v.y * inv * g.y, v.z * inv * g.z, v.w * inv * g.w));
    }
}

template <bool XF32>
__global__ void __launch_bounds__(kRowThreads) rows_normadd_kernel(const void* __restrict__ x,
                                                                  const float* __restrict__ w, float* __restrict__ h,
                                                                  int D, float scl) {
    __shared__ float red[kRowThreads / 32];
    const int D4 = D / 4;
    const size_t row4 = (size_t)blockIdx.x * D4;
    const float inv = row_inv_rms<XF32>(x, row4, D4, red);
    float4* h4 = reinterpret_cast<float4*>(h);
    for (int i = threadIdx.x; i < D4; i += kRowThreads) {
        const float4 v = ld4<XF32>(x, row4 + i), g = __ldg(reinterpret_cast<const float4*>(w) + i);
        float4 o = h4[row4 + i];
        o.x = (o.x + v.x * inv * g.x) * scl;
        o.y = (o.y + v.y * inv * g.y) * scl;
        o.z = (o.z + v.z * inv * g.z) * scl;
        o.w = (o.w + v.w * inv * g.w) * scl;
        h4[row4 + i] = o;
    }
}

__device__ __forceinline__ float gelu_tanh(float x) {
    // vk/gelumul.comp:8, the tanh approximation with the shader's constants
    return 0.5f * x * (1.0f + tanhf(0.7978845608028654f * (x + 0.044715f * x * x * x)));
}

template <bool XF32, bool YF32>
__global__ void __launch_bounds__(kRowThreads) gelumul_kernel(const void* __restrict__ gate, const void* __restrict__ up,
                                                             void* __restrict__ out, size_t n4) {
    const size_t stride = (size_t)gridDim.x * blockDim.x;
    for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n4; i += stride) {
        const float4 g = ld4<XF32>(gate, i), u = ld4<XF32>(up, i);
        st4<YF32>(out, i, make_float4(gelu_tanh(g.x) * u.x, gelu_tanh(g.y) * u.y, gelu_tanh(g.z) * u.z,
                                      gelu_tanh(g.w) * u.w));
    }
}

// ------------------------------------------------------------------ residual norm with int8 output
// h' = (h + x rsqrt(mean(x^2) + eps) w_post) scl,  t = h' w,  y = t rsqrt(mean(h'^2) + eps),
// sa = max(max|y| / 127, 1e-12),  A8 = rne(y / sa).
// The second norm's factor is one positive number r per row, so max|y| = r max|t|, and y / sa is t (127 / max|t|):
// the maximum and the sum of squares come out of the same reduction, and r enters sa alone.  A row stays in
// registers between the two reductions, so HBM sees x, h, h', A8 once: 11 bytes an element with f16 x.
struct NormI8Args {
    const void* x;         // null: h' = h scl
    const float* w_post;   // null: h' = (h + x) scl
    const float* h;
    float* h_out;          // may be h; null: not stored
    const float* w;
    int8_t* a8;
    float* sa;
    int D;
    float scl;
};

// the block's sum of s and maximum of m
__device__ __forceinline__ void block_sum_max(float& s, float& m, float2* red) {
    #pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) red[threadIdx.x >> 5] = make_float2(s, m);
    __syncthreads();
    const float2 v = lane < warps ? red[lane] : make_float2(0.f, 0.f);
    s = v.x;
    m = v.y;
    #pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
}

// Eight elements: f32 as one 32-byte access, f16 as one of 16
struct F8 {
    float v[8];
};
__device__ __forceinline__ F8 ld8(const float* p) {
    F8 r;
    asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(r.v[0]), "=f"(r.v[1]), "=f"(r.v[2]), "=f"(r.v[3]), "=f"(r.v[4]), "=f"(r.v[5]), "=f"(r.v[6]),
                   "=f"(r.v[7])
                 : "l"(p));
    return r;
}
__device__ __forceinline__ void st8(float* p, const F8& r) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(r.v[0]), "f"(r.v[1]), "f"(r.v[2]),
                 "f"(r.v[3]), "f"(r.v[4]), "f"(r.v[5]), "f"(r.v[6]), "f"(r.v[7])
                 : "memory");
}
// x as it lies in memory: the f16 form is half the registers while the sum of squares is on its way
template <bool F32>
struct X8;
template <>
struct X8<true> {
    F8 r;
    __device__ __forceinline__ void load(const void* p, size_t e) { r = ld8(reinterpret_cast<const float*>(p) + e); }
    __device__ __forceinline__ float at(int i) const { return r.v[i]; }
    __device__ __forceinline__ void zero() {
        #pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = 0.f;
    }
};
template <>
struct X8<false> {
    uint32_t r[4];
    __device__ __forceinline__ void load(const void* p, size_t e) {
        const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(p) + e);
        r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w;
    }
    __device__ __forceinline__ float at(int i) const { return i & 1 ? h_hi(r[i / 2]) : h_lo(r[i / 2]); }
    __device__ __forceinline__ void zero() { r[0] = r[1] = r[2] = r[3] = 0u; }
};

// codes: round-half-even of t * inv within [-127, 127], four to a word (vk/cast_i8.comp:18)
__device__ __forceinline__ uint2 quant8(const F8& t, float inv) {
    uint32_t w[2];
    #pragma unroll
    for (int k = 0; k < 2; k++) {
        w[k] = 0;
        #pragma unroll
        for (int i = 0; i < 4; i++)
            w[k] |= (uint32_t)(max(-127, min(127, __float2int_rn(t.v[4 * k + i] * inv))) & 0xff) << (8 * i);
    }
    return make_uint2(w[0], w[1]);
}

// sa of the row, and the factor from t to the codes
__device__ __forceinline__ float row_scale(float sum, float top, int D, float& inv) {
    const float r = rsqrtf(sum / (float)D + kRowEps);
    const float s = top * r / 127.0f;
    inv = s > 1e-12f ? 127.0f / top : r * 1e12f;
    return fmaxf(s, 1e-12f);
}

// h' of eight elements (h, x as they are, r the first norm's factor)
template <bool XF32>
__device__ __forceinline__ void update8(F8& h, const X8<XF32>& x, float r, const float* w_post, int e, float scl) {
    F8 g;
    if (w_post) g = ld8(w_post + e);
    #pragma unroll
    for (int i = 0; i < 8; i++) h.v[i] = (h.v[i] + (w_post ? x.at(i) * r * g.v[i] : x.at(i))) * scl;
}

// t = h' w, its largest magnitude and h' 's sum of squares
__device__ __forceinline__ void weigh8(F8& h, const float* w, int e, float& s, float& m) {
    const F8 g = ld8(w + e);
    #pragma unroll
    for (int i = 0; i < 8; i++) {
        s = fmaf(h.v[i], h.v[i], s);
        h.v[i] *= g.v[i];
        m = fmaxf(m, fabsf(h.v[i]));
    }
}

// NV groups of eight elements per thread; blockDim.x * NV >= D / 8
template <bool XF32, int NV>
__global__ void __launch_bounds__(NV > 2 ? 512 : 1024) rows_normadd_i8_kernel(const NormI8Args a) {
    __shared__ float2 red[2][32];
    const size_t row = (size_t)blockIdx.x * a.D;
    F8 h[NV];
    X8<XF32> x[NV];
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int e = 8 * (threadIdx.x + k * blockDim.x);
        x[k].zero();
        if (e < a.D) {
            if (a.x) x[k].load(a.x, row + e);
            h[k] = ld8(a.h + row + e);
        }
    }
    float s = 0.f, m = 0.f, r = 1.f;
    const float* w_post = a.x ? a.w_post : nullptr;
    if (w_post) {
        #pragma unroll
        for (int k = 0; k < NV; k++)
            #pragma unroll
            for (int i = 0; i < 8; i++) s = fmaf(x[k].at(i), x[k].at(i), s);
        block_sum_max(s, m, red[0]);
        r = rsqrtf(s / (float)a.D + kRowEps);
    }
    s = m = 0.f;
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int e = 8 * (threadIdx.x + k * blockDim.x);
        if (e < a.D) {
            update8<XF32>(h[k], x[k], r, w_post, e, a.scl);
            if (a.h_out) st8(a.h_out + row + e, h[k]);
            weigh8(h[k], a.w, e, s, m);
        }
    }
    block_sum_max(s, m, red[1]);
    float inv;
    const float sa = row_scale(s, m, a.D, inv);
    if (threadIdx.x == 0) a.sa[blockIdx.x] = sa;
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int e = 8 * (threadIdx.x + k * blockDim.x);
        if (e < a.D) *reinterpret_cast<uint2*>(a.a8 + row + e) = quant8(h[k], inv);
    }
}

// rows longer than the registers of a block: three passes, the later ones from L2
template <bool XF32>
__global__ void __launch_bounds__(1024) rows_normadd_i8_long_kernel(const NormI8Args a) {
    __shared__ float2 red[2][32];
    const size_t row = (size_t)blockIdx.x * a.D;
    const float* w_post = a.x ? a.w_post : nullptr;
    X8<XF32> x;
    x.zero();
    float s = 0.f, m = 0.f, r = 1.f;
    if (w_post) {
        for (int e = 8 * threadIdx.x; e < a.D; e += 8 * blockDim.x) {
            x.load(a.x, row + e);
            #pragma unroll
            for (int i = 0; i < 8; i++) s = fmaf(x.at(i), x.at(i), s);
        }
        block_sum_max(s, m, red[0]);
        r = rsqrtf(s / (float)a.D + kRowEps);
    }
    // t of a group; the first pass stores h', and the second one, for which h may be gone, reads it back
    auto group = [&](int e, bool first, float& sum, float& top) {
        F8 h;
        if (first || !a.h_out) {
            h = ld8(a.h + row + e);
            if (a.x) x.load(a.x, row + e);
            update8<XF32>(h, x, r, w_post, e, a.scl);
            if (a.h_out) st8(a.h_out + row + e, h);
        } else {
            h = ld8(a.h_out + row + e);
        }
        weigh8(h, a.w, e, sum, top);
        return h;
    };
    s = m = 0.f;
    for (int e = 8 * threadIdx.x; e < a.D; e += 8 * blockDim.x) group(e, true, s, m);
    block_sum_max(s, m, red[1]);
    float inv, s1 = 0.f, m1 = 0.f;
    const float sa = row_scale(s, m, a.D, inv);
    if (threadIdx.x == 0) a.sa[blockIdx.x] = sa;
    for (int e = 8 * threadIdx.x; e < a.D; e += 8 * blockDim.x)
        *reinterpret_cast<uint2*>(a.a8 + row + e) = quant8(group(e, false, s1, m1), inv);
}

// Threads and groups per thread.  Few rows (latency): as many threads as there are groups, up to a block.  Many rows:
// three groups per thread, so that several blocks share an SM and one's loads cover another's reductions; 8,192 rows of
// 3,840 f16: 57 us (6.1 TB/s, 0.93 of the measured copy rate), against 63 us with two groups and 95 us with one
// 16-byte group of four per thread.  Up to 256 groups one each is as fast (8,192 x 1,024: 18.5 us against 18.8).
template <bool XF32>
static void launch_normadd_i8(const NormI8Args& a, int M, int sms, cudaStream_t s) {
    const int groups = a.D / 8;
    const int nv = groups <= 256 ? 1 : M <= 2 * sms && groups <= 1024 ? 1 : groups <= 768 ? 3 : groups <= 2048 ? 4 : 0;
    const int threads = nv ? ((groups + nv - 1) / nv + 31) / 32 * 32 : 1024;
    switch (nv) {
        case 1: rows_normadd_i8_kernel<XF32, 1><<<M, threads, 0, s>>>(a); break;
        case 3: rows_normadd_i8_kernel<XF32, 3><<<M, threads, 0, s>>>(a); break;
        case 4: rows_normadd_i8_kernel<XF32, 4><<<M, threads, 0, s>>>(a); break;
        default: rows_normadd_i8_long_kernel<XF32><<<M, threads, 0, s>>>(a);
    }
}

static bool dt_ok(int dt) { return dt == G4B_DT_F32 || dt == G4B_DT_F16; }

}  // namespace g4b

using namespace g4b;

extern "C" {

int g4b_rows_rmsnorm(const void* x, int x_dtype, const float* w, void* y, int y_dtype, int M, int D,
                     g4b_stream_t stream) {
    G4B_ENTRY("rows_rmsnorm");
    G4B_REQUIRE(x && w && y, G4B_E_ARG, "rows_rmsnorm: NULL pointer");
    G4B_REQUIRE(dt_ok(x_dtype) && dt_ok(y_dtype), G4B_E_ARG, "rows_rmsnorm: bad dtype %d / %d", x_dtype, y_dtype);
    G4B_REQUIRE(M >= 1 && M <= 0x7fffffff && D >= 4 && D % 4 == 0, G4B_E_SHAPE,
                "rows_rmsnorm: M=%d D=%d (D a multiple of 4)", M, D);
    G4B_REQUIRE(aligned16(x) && aligned16(w) && aligned16(y), G4B_E_ALIGN,
                "rows_rmsnorm: x, w and y must be 16-byte aligned");
    int st = check_device(nullptr);
    if (st != G4B_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const bool xf = x_dtype == G4B_DT_F32, yf = y_dtype == G4B_DT_F32;
    if (xf && yf) rows_rmsnorm_kernel<true, true><<<M, kRowThreads, 0, s>>>(x, w, y, D);
    else if (xf) rows_rmsnorm_kernel<true, false><<<M, kRowThreads, 0, s>>>(x, w, y, D);
    else if (yf) rows_rmsnorm_kernel<false, true><<<M, kRowThreads, 0, s>>>(x, w, y, D);
    else rows_rmsnorm_kernel<false, false><<<M, kRowThreads, 0, s>>>(x, w, y, D);
    count_launch();
    return launch_status("rows_rmsnorm");
}

int g4b_rows_normadd(const void* x, int x_dtype, const float* w, float* h, int M, int D, float scl,
                     g4b_stream_t stream) {
    G4B_ENTRY("rows_normadd");
    G4B_REQUIRE(x && w && h, G4B_E_ARG, "rows_normadd: NULL pointer");
    G4B_REQUIRE(dt_ok(x_dtype), G4B_E_ARG, "rows_normadd: bad dtype %d", x_dtype);
    G4B_REQUIRE(M >= 1 && D >= 4 && D % 4 == 0, G4B_E_SHAPE, "rows_normadd: M=%d D=%d (D a multiple of 4)", M, D);
    G4B_REQUIRE(aligned16(x) && aligned16(w) && aligned16(h), G4B_E_ALIGN,
                "rows_normadd: x, w and h must be 16-byte aligned");
    int st = check_device(nullptr);
    if (st != G4B_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (x_dtype == G4B_DT_F32) rows_normadd_kernel<true><<<M, kRowThreads, 0, s>>>(x, w, h, D, scl);
    else rows_normadd_kernel<false><<<M, kRowThreads, 0, s>>>(x, w, h, D, scl);
    count_launch();
    return launch_status("rows_normadd");
}

int g4b_gelumul(const void* gate, const void* up, int dtype, void* out, int out_dtype, size_t n,
                g4b_stream_t stream) {
    G4B_ENTRY("gelumul");
    G4B_REQUIRE(gate && up && out, G4B_E_ARG, "gelumul: NULL pointer");
    G4B_REQUIRE(dt_ok(dtype) && dt_ok(out_dtype), G4B_E_ARG, "gelumul: bad dtype %d / %d", dtype, out_dtype);
    G4B_REQUIRE(n >= 4 && n % 4 == 0, G4B_E_SHAPE, "gelumul: n=%zu (a multiple of 4)", n);
    G4B_REQUIRE(aligned16(gate) && aligned16(up) && aligned16(out), G4B_E_ALIGN,
                "gelumul: gate, up and out must be 16-byte aligned");
    int sms = 148;
    int st = check_device(&sms);
    if (st != G4B_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const size_t n4 = n / 4;
    const int grid = (int)std::min<size_t>((n4 + kRowThreads - 1) / kRowThreads, (size_t)sms * 8);
    const bool xf = dtype == G4B_DT_F32, yf = out_dtype == G4B_DT_F32;
    if (xf && yf) gelumul_kernel<true, true><<<grid, kRowThreads, 0, s>>>(gate, up, out, n4);
    else if (xf) gelumul_kernel<true, false><<<grid, kRowThreads, 0, s>>>(gate, up, out, n4);
    else if (yf) gelumul_kernel<false, true><<<grid, kRowThreads, 0, s>>>(gate, up, out, n4);
    else gelumul_kernel<false, false><<<grid, kRowThreads, 0, s>>>(gate, up, out, n4);
    count_launch();
    return launch_status("gelumul");
}

int g4b_rows_normadd_i8(const void* x, int x_dtype, const float* w_post, const float* h, float* h_out, float scl,
                        const float* w, int8_t* A8, float* sa, int M, int D, g4b_stream_t stream) {
    G4B_ENTRY("rows_normadd_i8");
    G4B_REQUIRE(h && w && A8 && sa, G4B_E_ARG, "rows_normadd_i8: NULL pointer");
    G4B_REQUIRE(x || !w_post, G4B_E_ARG, "rows_normadd_i8: w_post without x");
    G4B_REQUIRE(!x || dt_ok(x_dtype), G4B_E_ARG, "rows_normadd_i8: bad dtype %d", x_dtype);
    // (the loops over a long row count in 32 bits, a block's step beyond its end)
    G4B_REQUIRE(M >= 1 && D >= 16 && D % 16 == 0 && D <= 1 << 30, G4B_E_SHAPE,
                "rows_normadd_i8: M=%d D=%d (D a multiple of 16, at most 2^30)", M, D);
    const size_t n = (size_t)M * D;
    G4B_REQUIRE(!h_out || h_out == h || !rows_overlap(flat(h_out, 4 * n), flat(h, 4 * n)), G4B_E_ARG,
                "rows_normadd_i8: h_out overlaps h without being h");
    const auto aligned32 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; };
    G4B_REQUIRE(aligned32(x) && aligned32(w_post) && aligned32(h) && aligned32(h_out) && aligned32(w) && aligned16(A8) &&
                    ((uintptr_t)sa & 3u) == 0,
                G4B_E_ALIGN, "rows_normadd_i8: x, the weights, h and h_out must be 32-byte aligned, A8 16-byte, sa 4-byte");
    const Rows read[] = {flat(x, n * (x_dtype == G4B_DT_F32 ? 4 : 2)), flat(w_post, 4 * (size_t)D), flat(w, 4 * (size_t)D)};
    const Rows codes = flat(A8, n), scales = flat(sa, 4 * (size_t)M);
    bool clash = rows_overlap(codes, scales);
    for (const Rows& r : {flat(h, 4 * n), flat(h_out, 4 * n)}) clash |= rows_overlap(r, codes) || rows_overlap(r, scales);
    for (const Rows& r : read) clash |= rows_overlap(r, codes) || rows_overlap(r, scales) || rows_overlap(r, flat(h_out, 4 * n));
    G4B_REQUIRE(!clash, G4B_E_ARG, "rows_normadd_i8: what it writes overlaps what it reads");
    int sms = 148;
    int st = check_device(&sms);
    if (st != G4B_OK) return st;
    NormI8Args a{x, w_post, h, h_out, w, A8, sa, D, scl};
    if (x && x_dtype == G4B_DT_F32) launch_normadd_i8<true>(a, M, sms, reinterpret_cast<cudaStream_t>(stream));
    else launch_normadd_i8<false>(a, M, sms, reinterpret_cast<cudaStream_t>(stream));
    count_launch();
    return launch_status("rows_normadd_i8");
}

}  // extern "C"
