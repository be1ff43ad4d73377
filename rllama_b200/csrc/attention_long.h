// Device helpers shared by the long-context attention kernels: the visible set, cache rows as f32, the plain form of a row.
#pragma once

#include <algorithm>
#include <cfloat>

#include "cache4.h"
#include "internal.h"

namespace attn_long {

struct Run {
    int s, l, len;  // first run [0, s), second [l, l + len - s)
    __device__ __forceinline__ int at(int v) const { return v < s ? v : v - s + l; }
};
__device__ __forceinline__ int window_low(const AttnLongArgs& a, int p) { return max(0, p + 1 - a.window); }
__device__ __forceinline__ Run visible_run(const AttnLongArgs& a, int p0, int p1) {
    Run r;
    r.l = window_low(a, p0);
    r.s = min(a.sinks, r.l);
    r.len = r.s + p1 + 1 - r.l;
    return r;
}
__device__ __forceinline__ bool visible(const AttnLongArgs& a, int p, int t) { return t <= p && (t >= window_low(a, p) || t < a.sinks); }

// HD / 32 neighbouring values of a cache row, as f32.
template <int KIND, int HD> __device__ __forceinline__ void load_row(const void* base, const __half* scales, int64_t row, int lane, float (&x)[HD / 32]) {
    constexpr int N = HD / 32;
    if constexpr (KIND == CACHE_F32) {
        const float* p = reinterpret_cast<const float*>(base) + row * HD + lane * N;
        if constexpr (N == 4) { const float4 v = *reinterpret_cast<const float4*>(p); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
        else { const float2 v = *reinterpret_cast<const float2*>(p); x[0] = v.x; x[1] = v.y; }
    } else {
        __half2 h[N / 2];
        if constexpr (KIND == CACHE_F16) {
            const __half* p = reinterpret_cast<const __half*>(base) + row * HD + lane * N;
            if constexpr (N == 4) *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(p);
            else *reinterpret_cast<uint32_t*>(h) = *reinterpret_cast<const uint32_t*>(p);
        } else {
            constexpr int G = HD / kQ4Group;
            const int e = lane * N;
            const uint32_t w = reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(base) + row * (HD / 2))[q4_word(e, G)];
            const __half2 d = __half2half2(scales[row * G + e / kQ4Group]);
#pragma unroll
            for (int j = 0; j < N / 2; j++) h[j] = __hmul2(q4_pair(w, (e % 8) / 2 + j), d);
        }
#pragma unroll
        for (int j = 0; j < N / 2; j++) {
            const float2 f = __half22float2(h[j]);
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
        }
    }
}

// The plain form of a row, by one warp: lanes over head_dim, one position after the other. Maximum m, sum l, unnormalised result o.
template <int KIND, int HD> struct PlainRow {
    static constexpr int N = HD / 32;
    float q[N], o[N] = {}, m = -FLT_MAX, l = 0.f;
    __device__ __forceinline__ PlainRow(const AttnLongArgs& a, int i, int head, int lane) {
        const float c2 = rsqrtf((float)HD) * 1.4426950408889634f;
#pragma unroll
        for (int e = 0; e < N; e++) q[e] = a.q[i * a.q_ld + head * HD + lane * N + e] * c2;
    }
    __device__ __forceinline__ void see(const AttnLongArgs& a, int64_t row, int lane) {   // the position at that row of the cache
        float k[N], x[N], s = 0.f;
        load_row<KIND, HD>(a.k, a.k_scale, row, lane, k);
        load_row<KIND, HD>(a.v, a.v_scale, row, lane, x);
#pragma unroll
        for (int e = 0; e < N; e++) s = fmaf(q[e], k[e], s);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float m_new = fmaxf(m, s), w = exp2f(s - m_new), scale = exp2f(m - m_new);
        l = l * scale + w;
#pragma unroll
        for (int e = 0; e < N; e++) o[e] = fmaf(o[e], scale, w * x[e]);
        m = m_new;
    }
};

__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
// A mean of f16 values as f16. Weights that were rounded up may put a mean of values next to the largest f16 beyond it (up to 65504 (1 + 2^-11)), and only
// an infinity that the row sees may make one.
constexpr float kMaxF16 = 65504.f, kInfF16 = 65520.f;   // (from there on a rounded f16 is infinite)
__device__ __forceinline__ float within_f16(float v) { return fabsf(v) <= FLT_MAX ? fminf(fmaxf(v, -kMaxF16), kMaxF16) : v; }
__device__ __forceinline__ void store_out(__half* p, float v) { *p = __float2half_rn(within_f16(v)); }
__device__ __forceinline__ __half2 mean_f16(float x, float y) {
    if (fmaxf(fabsf(x), fabsf(y)) >= kInfF16) { x = within_f16(x); y = within_f16(y); }
    return __floats2half2_rn(x, y);
}

constexpr uint32_t kWaitLimit = 1u << 22;
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t mbar_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok;
}
// Bounded wait; false when it ran out or the CTA already gave up.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* dead, int* err) {
    for (uint32_t i = 0; i < kWaitLimit; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 63u && *dead) return false;
    }
    *dead = 1;
    *reinterpret_cast<volatile int*>(err) = 4;
    return false;
}
// The same for a whole warp, with one answer for all of its lanes (they go on together or not at all). What is there
// already costs one look (512-row 4-bit chunk 150 us with the loop alone, 142 with it).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* dead, int* err) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, dead, err));
}
// Waits, with the same limit, for work of the CTA's own that is in flight, whether or not the CTA gave up.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kWaitLimit && !mbar_try_wait(bar, parity); i++) {}
}
// |x| into a running maximum; a NaN stays.
__device__ __forceinline__ void max_abs_nan(float& top, float x) { asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x))); }
// Whether a row of sum l, unnormalised results up to o_top in magnitude and maximum m has to be computed again from what it sees alone: a NaN that the
// sum does not have may come from a position that the row does not see, times weight zero. Anything else that is not finite comes from what it sees, and is
// the result, unless the scores are so large (beyond 2^20) that a weight may have left the range of f16 or f32. (|m| = FLT_MAX: no score counted yet.)
__device__ __forceinline__ bool row_is_suspect(float l, float o_top, float m) {
    if (fabsf(m) > 0x1p20f && fabsf(m) < FLT_MAX) return !(l <= FLT_MAX && o_top <= FLT_MAX);
    return l == l && o_top != o_top;
}
__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace attn_long

// How many parts the positions of a row block are split into, and whether the parts are joined by a second kernel.
struct AttnSplit {
    int n;
    bool records;
};
// Splits whose records take up to 64 MB: scratch is memory that the caller's caches do not get.
inline int64_t record_limit(const AttnLongArgs& a) { return std::max<int64_t>(1, (64ll << 20) / ((int64_t)a.n * a.heads * (a.hd * 4 + 8))); }

// attention_long_few.cu
AttnSplit attn_long_few_splits(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a);
double attn_long_few_us(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a, AttnSplit s);
int launch_attn_long_few(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a);
// attention_long_f32.cu
int attn_long_f32_splits(rlb_ctx* ctx, const AttnLongArgs& a);
double attn_long_f32_us(rlb_ctx* ctx, const AttnLongArgs& a, int splits);   // the time it will take, roughly
int launch_attn_long_f32(rlb_ctx* ctx, const AttnLongArgs& a);
// attention_long_tc.cu
int attn_long_tc_splits(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a);
double attn_long_tc_us(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a, int splits);
int launch_attn_long_tc(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a);
