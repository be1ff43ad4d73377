// The way of q, k and v rows from their projection into attention, as one op: optional RMSNorm of every q and k head
// (RMSNorm::forward, src/transformer.rs:476-480, over head_dim), the rotation of neighbouring pairs (apply_rotary_emb,
// src/transformer.rs:823-856) and the cache write loop (:751-761).
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * gain            (only with gains)
//   (a, b) -> (a cos - b sin, a sin + b cos)              pairs (2j, 2j+1), angle = position * 10000^(-2j / head_dim)
//
// All of it is f32; a cache row is rounded once, to the cache's dtype.
//
// Every value is read and written once, so memory is the bound: 1792 rows of 64 heads and 64 K/V heads of 128 into f16 caches, with the norm, take 51 us
// a call, 5.7 TB/s (47 in a graph; one row a thread at a time 63; two or eight no faster than four; streaming loads and stores neither). Instructions count
// beside it: with a reduction over the warp, a square root and a division for every row it was 57. A token's row is 2 us in a graph, and a call's 5 us.
#include "internal.h"

#include <algorithm>
#include <cmath>
#include <new>

namespace {

struct RotateArgs {
    const float* q; const float* k; const float* v;
    float* q_out;
    int64_t q_ld, k_ld, v_ld, qo_ld;
    const float* q_gain; const float* k_gain;  // null: no norm
    const float* table; int64_t table_ld;      // row of a position: (cos, sin) of pair 0, 1, ...
    void* kcache; void* vcache;
    int n, heads, kv_heads, max_seq, start;
    float eps;
};

template <int N> struct Vec;
template <> struct Vec<4> { typedef float4 T; };
template <> struct Vec<2> { typedef float2 T; };

template <typename CT, int N> __device__ __forceinline__ void store_cache(CT* p, const float (&x)[N]) {
    if constexpr (sizeof(CT) == 2) {
        __half2 h[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; e++) h[e] = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
        if constexpr (N == 4) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
        else *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(h);
    } else {
        *reinterpret_cast<typename Vec<N>::T*>(p) = *reinterpret_cast<const typename Vec<N>::T*>(x);
    }
}

// grid (slots / 8, tokens): a warp per slot (the q heads, the k heads, the v heads) and U tokens, whose loads are all in flight. A lane
// holds HD / 32 neighbouring values, i.e. whole pairs, and the norm's sum is one reduction over the warp.
constexpr int U = 4;   // (the norm's sums are dealt to the lanes four rows at a time)

template <typename CT, int HD>
__global__ void __launch_bounds__(256) norm_rope_append_kernel(const __grid_constant__ RotateArgs a) {
    constexpr int N = HD / 32;
    typedef typename Vec<N>::T V;
    const int slot = blockIdx.x * 8 + (threadIdx.x >> 5), c = (threadIdx.x & 31) * N;
    if (slot >= a.heads + 2 * a.kv_heads) return;
    const int kind = slot < a.heads ? 0 : slot < a.heads + a.kv_heads ? 1 : 2;
    const int head = kind == 0 ? slot : kind == 1 ? slot - a.heads : slot - a.heads - a.kv_heads;
    const float* src = (kind == 0 ? a.q : kind == 1 ? a.k : a.v) + head * HD + c;
    const int64_t ld = kind == 0 ? a.q_ld : kind == 1 ? a.k_ld : a.v_ld;
    const float* gain = kind == 0 ? a.q_gain : kind == 1 ? a.k_gain : nullptr;
    float g[N];
    if (gain) *reinterpret_cast<V*>(g) = *reinterpret_cast<const V*>(gain + c);
    CT* cache = reinterpret_cast<CT*>(kind == 2 ? a.vcache : a.kcache) + ((int64_t)head * a.max_seq + a.start) * HD + c;
    const int lane = threadIdx.x & 31;
    for (int i0 = blockIdx.y * U; i0 < a.n; i0 += gridDim.y * U) {
        const int last = a.n - 1 - i0;   // of the U rows
        const float *p = src + i0 * ld, *t = a.table + (a.start + i0) * a.table_ld + c;
        float x[U][N], f[U][N];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int y = min(u, last);
            *reinterpret_cast<V*>(x[u]) = *reinterpret_cast<const V*>(p + y * ld);
            if (kind != 2) *reinterpret_cast<V*>(f[u]) = *reinterpret_cast<const V*>(t + y * a.table_ld);
        }
        if (kind != 2) {
            if (gain) {
                // The rows' sums of squares, four at a time: lanes hand on half of the rows that they hold until they hold one, eight lanes a row. The order of the
                // additions (values 4 apart, with head_dim 128 then 32, or else 2 and 4; then 8, 16 and the row's halves) is that of cache4.cu, whose
                // rotation has the same bits.
                float ss[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    ss[u] = 0.f;
#pragma unroll
                    for (int e = 0; e < N; e++) ss[u] = fmaf(x[u][e], x[u][e], ss[u]);
                }
                constexpr int SECOND = N == 4 ? 8 : 2;
                const bool up = lane & 1, odd = lane & SECOND;
                float s0 = (up ? ss[2] : ss[0]) + __shfl_xor_sync(0xffffffffu, up ? ss[0] : ss[2], 1);
                float s1 = (up ? ss[3] : ss[1]) + __shfl_xor_sync(0xffffffffu, up ? ss[1] : ss[3], 1);
                s0 = (odd ? s1 : s0) + __shfl_xor_sync(0xffffffffu, odd ? s0 : s1, SECOND);
                s0 += __shfl_xor_sync(0xffffffffu, s0, N == 4 ? 2 : 4);
                s0 += __shfl_xor_sync(0xffffffffu, s0, N == 4 ? 4 : 8);
                s0 += __shfl_xor_sync(0xffffffffu, s0, 16);
                const float s = 1.0f / sqrtf(s0 / (float)HD + a.eps);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const float su = __shfl_sync(0xffffffffu, s, (u >> 1) + (u & 1) * SECOND);
#pragma unroll
                    for (int e = 0; e < N; e++) x[u][e] = x[u][e] * su * g[e];
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const float x0 = x[u][e], x1 = x[u][e + 1];
                    x[u][e] = __fsub_rn(__fmul_rn(x0, f[u][e]), __fmul_rn(x1, f[u][e + 1]));
                    x[u][e + 1] = __fadd_rn(__fmul_rn(x0, f[u][e + 1]), __fmul_rn(x1, f[u][e]));
                }
        }
        if (kind == 0) {
            float* dst = a.q_out + i0 * a.qo_ld + head * HD + c;
#pragma unroll
            for (int u = 0; u < U; u++)
                if (u <= last) *reinterpret_cast<V*>(dst + u * a.qo_ld) = *reinterpret_cast<const V*>(x[u]);
        } else {
#pragma unroll
            for (int u = 0; u < U; u++)
                if (u <= last) store_cache<CT, N>(cache + (int64_t)i0 * HD + u * HD, x[u]);
        }
    }
}

template <typename CT>
void launch(const RotateArgs& a, int hd, cudaStream_t s) {
    const dim3 grid((unsigned)((a.heads + 2 * a.kv_heads + 7) / 8), (unsigned)std::min((a.n + U - 1) / U, 65535));
    if (hd == 128) norm_rope_append_kernel<CT, 128><<<grid, 256, 0, s>>>(a);
    else norm_rope_append_kernel<CT, 64><<<grid, 256, 0, s>>>(a);
}

int check_gain(const rlb_tensor* g, const rlb_tensor* like, int64_t hd) {
    if (!g) return RLB_OK;
    RLB_TRY(same_ctx(g, like));
    if (g->dtype != RLB_F32 || g->rows != 1 || g->cols != hd) return rlb_fail(RLB_ERR_INVALID, "norm_rope_append: a gain must be 1 x head_dim f32");
    return RLB_OK;
}

}  // namespace

extern "C" int rlb_rope_table(rlb_ctx* ctx, int32_t max_seq_len, int32_t head_dim, rlb_tensor** out) {
    if (!ctx || !out) return rlb_fail(RLB_ERR_INVALID, "rlb_rope_table: null pointer");
    *out = nullptr;
    if (max_seq_len < 1 || head_dim < 4 || head_dim % 4 != 0)
        return rlb_fail(RLB_ERR_INVALID, "rlb_rope_table: bad max_seq_len %d or head_dim %d (a multiple of 4)", max_seq_len, head_dim);
    DeviceScope dev(ctx->device);
    if (ctx_capturing(ctx)) return rlb_fail(RLB_ERR_STATE, "rlb_rope_table allocates: it cannot be captured into a graph");
    // compute_freqs_cis (src/transformer.rs:858-885): f64 angles, narrowed to f32 where they are applied
    float* tab = new (std::nothrow) float[(size_t)max_seq_len * head_dim];
    if (!tab) return rlb_fail(RLB_ERR_OOM, "rlb_rope_table: out of host memory");
    for (int i = 0; i < head_dim / 2; i++) {
        const double freq = 1.0 / pow(10000.0, (double)i * 2.0 / (double)head_dim);
        for (int pos = 0; pos < max_seq_len; pos++) {
            const double ang = freq * (double)pos;
            tab[(size_t)pos * head_dim + 2 * i] = (float)cos(ang);
            tab[(size_t)pos * head_dim + 2 * i + 1] = (float)sin(ang);
        }
    }
    int s = dev.err == cudaSuccess ? RLB_OK : rlb_fail(RLB_ERR_CUDA, "rlb_rope_table: %s", cudaGetErrorString(dev.err));
    if (s == RLB_OK) s = rlb_tensor_upload(ctx, tab, max_seq_len, head_dim, head_dim, RLB_F32, out);
    if (s == RLB_OK) s = rlb_tensor_wait(*out);
    if (s != RLB_OK && *out) {
        rlb_tensor_free(*out);
        *out = nullptr;
    }
    delete[] tab;
    return s;
}

extern "C" int rlb_norm_rope_append(rlb_tensor* q_out, rlb_tensor* kcache, rlb_tensor* vcache, const rlb_tensor* q, const rlb_tensor* k,
                                    const rlb_tensor* v, const rlb_tensor* q_gain, const rlb_tensor* k_gain, float eps, const rlb_tensor* rope,
                                    int32_t heads, int32_t kv_heads, int32_t max_seq_len, int32_t start_pos) {
    for (const rlb_tensor* t : {(const rlb_tensor*)kcache, (const rlb_tensor*)vcache, q, k, v, rope}) RLB_TRY(same_ctx(q_out, t));
    const int64_t n = q->rows, hd = kcache->cols;
    RLB_TRY(check_gain(q_gain, q_out, hd));
    RLB_TRY(check_gain(k_gain, q_out, hd));
    if (heads < 1 || kv_heads < 1 || max_seq_len < 1 || start_pos < 0 || start_pos + n > max_seq_len)
        return rlb_fail(RLB_ERR_INVALID, "norm_rope_append: bad heads %d, kv_heads %d, max_seq_len %d, start_pos %d or %lld rows", heads, kv_heads,
                        max_seq_len, start_pos, (long long)n);
    if (hd != 64 && hd != 128) return rlb_fail(RLB_ERR_INVALID, "norm_rope_append: head_dim %lld is not supported (64 or 128)", (long long)hd);
    if (kcache->cap != hd || vcache->cap != hd || vcache->cols != hd || kcache->rows != (int64_t)kv_heads * max_seq_len ||
        vcache->rows != kcache->rows || kcache->dtype != vcache->dtype)
        return rlb_fail(RLB_ERR_INVALID, "norm_rope_append: caches must be (kv_heads*max_seq_len) x head_dim without row padding");
    if (q->dtype != RLB_F32 || q->cols != heads * hd || q_out->dtype != RLB_F32 || q_out->rows != n || q_out->cols != q->cols)
        return rlb_fail(RLB_ERR_INVALID, "norm_rope_append: q and q_out must be n x heads*head_dim f32");
    if (k->dtype != RLB_F32 || k->rows != n || k->cols != kv_heads * hd || v->dtype != RLB_F32 || v->rows != n || v->cols != k->cols)
        return rlb_fail(RLB_ERR_INVALID, "norm_rope_append: k and v must be n x kv_heads*head_dim f32");
    if (std::max(q->cols, k->cols) > kMaxColumns)
        return rlb_fail(RLB_ERR_LIMIT, "norm_rope_append: rows of %lld columns are more than %lld", (long long)std::max(q->cols, k->cols), (long long)kMaxColumns);
    if (rope->dtype != RLB_F32 || rope->cols != hd || rope->rows < start_pos + n)
        return rlb_fail(RLB_ERR_INVALID, "norm_rope_append: the rope table must be f32, head_dim wide and cover position %lld", (long long)(start_pos + n - 1));
    if (!(eps >= 0.f)) return rlb_fail(RLB_ERR_INVALID, "norm_rope_append: eps must not be negative");
    if (n == 0) return RLB_OK;
    rlb_ctx* ctx = q_out->ctx;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    DeviceScope dev(ctx->device);
    RLB_CUDA(dev.err);
    RotateArgs a;
    a.q = (const float*)q->d; a.k = (const float*)k->d; a.v = (const float*)v->d; a.q_out = (float*)q_out->d;
    a.q_ld = q->cap; a.k_ld = k->cap; a.v_ld = v->cap; a.qo_ld = q_out->cap;
    a.q_gain = q_gain ? (const float*)q_gain->d : nullptr; a.k_gain = k_gain ? (const float*)k_gain->d : nullptr;
    a.table = (const float*)rope->d; a.table_ld = rope->cap;
    a.kcache = kcache->d; a.vcache = vcache->d;
    a.n = (int)n; a.heads = heads; a.kv_heads = kv_heads; a.max_seq = max_seq_len; a.start = start_pos; a.eps = eps;
    if (kcache->dtype == RLB_F16) launch<__half>(a, (int)hd, ctx->stream);
    else launch<float>(a, (int)hd, ctx->stream);
    RLB_LAUNCH_CHECK();
    count_launch(ctx);
    RLB_TRY(tensor_mark_ready(q_out));
    RLB_TRY(tensor_mark_ready(kcache));
    return tensor_mark_ready(vcache);
}
