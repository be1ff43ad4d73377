// The 4-bit cache (format: cache4.h): creation, appending rows and reading them back. What the reference keeps in f16 or
// f32 per head (src/transformer.rs:129-160, the write loop :751-761) in 0.5625 bytes a value.
#include "cache4.h"
#include "internal.h"

#include <algorithm>
#include <new>

namespace {

__device__ __forceinline__ float max_nan(float x, float y) {   // a NaN wins
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__half>(const __half* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(h[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

struct AppendArgs {
    const void* src[3];  // K and V rows, and with the rotation q rows
    int64_t ld[3];
    uint8_t* codes[2];
    __half* scales[2];
    int kv_heads, max_seq, start, n;
    // with the rotation (what it computes: rotate.cu)
    float* q_out;
    int64_t qo_ld;
    const float* gain[3];      // of K and q heads; null: no norm
    const float* table;        // a position's row: (cos, sin) of pair 0, 1, ...
    int64_t table_ld;
    float eps;
    int heads;
};

// All kernels: a grid over heads, rows, and K and V (with the rotation also q, whose rows go through f32 to where the caller wants them). A thread
// takes the same block of eight values of every group of a head's row when it reads, which is a quarter of the row's codes side by side
// (cache4.h), and of half of the groups when it writes; four or eight threads make a row. No thread divides by a runtime size. (1792 rows of 64
// heads of 128, f32, written and read back: one word a thread, found by 64-bit division: 51 + 49 us; this: 27 + 14 us, of 20 + 11 that the bytes
// take; f16 rows 23 in a graph, where f32 rows are 23.5. A quarter row a thread in the append too: 28, as it leaves room for half of the warps; two rows a thread, or CTAs of 256: up to 10 us
// more.) With the rotation, 64 heads of q beside them: 49 us, 5.2 TB/s (a quarter row a thread: 51), with the norm 57, where the two ops one after the
// other take 51 + 27; 64 heads on 8, with the norm, 31; a token's row 3.3 us in a graph, and a call's 4.
constexpr int kThreads = 128;
template <int G> struct Words;   // a thread's words of a row, and their scales
template <> struct Words<4> { typedef uint4 T; typedef uint2 D; };
template <> struct Words<1> { typedef uint32_t T; typedef unsigned short D; };
template <> struct Words<2> { typedef uint2 T; typedef uint32_t D; };

// Normalises (with a gain) and rotates a thread's values of a head's row, which are whole pairs; eight neighbouring threads have the row.
template <int G> __device__ __forceinline__ void norm_rope(float (&y)[G][8], const float* gain, float eps, const float* turn) {
    if (gain) {
        // (the additions in the order of rotate.cu: runs of 2 G values, their neighbours in the group of eight, the other group, the row's other threads)
        constexpr int RUN = 2 * G, RUNS = 8 / RUN;
        float ss = 0.f;
#pragma unroll
        for (int g = 0; g < G; g++) {
            float part[RUNS];
#pragma unroll
            for (int r = 0; r < RUNS; r++) {
                part[r] = 0.f;
#pragma unroll
                for (int e = 0; e < RUN; e++) part[r] = fmaf(y[g][r * RUN + e], y[g][r * RUN + e], part[r]);
            }
            const float sum = RUNS == 2 ? part[0] + part[1] : (part[0] + part[1]) + (part[RUNS - 2] + part[RUNS - 1]);
            ss = g == 0 ? sum : ss + sum;
        }
        ss += __shfl_xor_sync(0xffffffffu, ss, 1);
        ss += __shfl_xor_sync(0xffffffffu, ss, 2);
        ss += __shfl_xor_sync(0xffffffffu, ss, 4);
        const float s = 1.0f / sqrtf(ss / (float)(2 * G * kQ4Group) + eps);
#pragma unroll
        for (int g = 0; g < G; g++) {
            float w[8];
            load8<float>(gain + g * kQ4Group, w);
#pragma unroll
            for (int e = 0; e < 8; e++) y[g][e] = y[g][e] * s * w[e];
        }
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
        float f[8];
        load8<float>(turn + g * kQ4Group, f);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float x0 = y[g][e], x1 = y[g][e + 1];
            y[g][e] = __fsub_rn(__fmul_rn(x0, f[e]), __fmul_rn(x1, f[e + 1]));
            y[g][e + 1] = __fadd_rn(__fmul_rn(x0, f[e + 1]), __fmul_rn(x1, f[e]));
        }
    }
}

template <typename T, int HD, bool ROTATE>
__global__ void __launch_bounds__(kThreads) append4_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int ALL = HD / kQ4Group, G = ALL / 2;   // groups of a row, of a thread
    const int x = blockIdx.x * kThreads + threadIdx.x, which = blockIdx.z, block = x & 3, half = x >> 2 & 1;
    const int threads = (which == 2 ? a.heads : a.kv_heads) * 8;
    if (ROTATE && blockIdx.x * kThreads >= threads) return;   // (the grid is as wide as the most heads need: 64 heads on 8 49 us with these CTAs, 31 without)
    const bool live = x < threads;   // (a row's eight threads are all live or none is)
    const int head = live ? x >> 3 : 0;
    const T* src = reinterpret_cast<const T*>(a.src[which]) + head * HD + half * (HD / 2) + block * 8;
    for (int i = blockIdx.y; i < a.n; i += gridDim.y) {
        float y[G][8];
#pragma unroll
        for (int g = 0; g < G; g++) load8<T>(src + i * a.ld[which] + g * kQ4Group, y[g]);
        if constexpr (ROTATE) {
            if (which != 1) norm_rope<G>(y, a.gain[which] ? a.gain[which] + half * (HD / 2) + block * 8 : nullptr, a.eps, a.table + (a.start + i) * a.table_ld + half * (HD / 2) + block * 8);
            if (which == 2) {
                float* dst = a.q_out + i * a.qo_ld + head * HD + half * (HD / 2) + block * 8;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    if (!live) break;
                    *reinterpret_cast<float4*>(dst + g * kQ4Group) = make_float4(y[g][0], y[g][1], y[g][2], y[g][3]);
                    *reinterpret_cast<float4*>(dst + g * kQ4Group + 4) = make_float4(y[g][4], y[g][5], y[g][6], y[g][7]);
                }
                continue;
            }
        }
        uint32_t w[G];
        __half d[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) m = max_nan(m, fabsf(y[g][e]));
            m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
            d[g] = m != m ? __ushort_as_half(0x7fff) : q4_scale(m);
            w[g] = q4_pack(y[g], __half2float(d[g]));
        }
        if (!live) continue;
        const int64_t row = (int64_t)head * a.max_seq + a.start + i;
        *reinterpret_cast<typename Words<G>::T*>(a.codes[which] + row * (HD / 2) + block * (HD / 8) + half * (HD / 16)) = *reinterpret_cast<const typename Words<G>::T*>(w);
        if (block == 0) *reinterpret_cast<typename Words<G>::D*>(a.scales[which] + row * ALL + half * G) = *reinterpret_cast<const typename Words<G>::D*>(d);
    }
}

struct ReadArgs {
    void* dst[2];
    int64_t ld[2];
    const uint8_t* codes[2];
    const __half* scales[2];
    int kv_heads, max_seq, start, n;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) read4_kernel(const __grid_constant__ ReadArgs a) {
    constexpr int G = HD / kQ4Group;
    const int x = blockIdx.x * kThreads + threadIdx.x, which = blockIdx.z, block = x & 3, head = x >> 2;
    if (x >= a.kv_heads * 4 || a.dst[which] == nullptr) return;
    const int64_t base = (int64_t)head * a.max_seq + a.start;
    for (int i = blockIdx.y; i < a.n; i += gridDim.y) {
        const int64_t row = base + i;
        uint32_t w[G];
        __half d[G];
        *reinterpret_cast<typename Words<G>::T*>(w) = *reinterpret_cast<const typename Words<G>::T*>(a.codes[which] + row * (HD / 2) + block * (HD / 8));
        *reinterpret_cast<typename Words<G>::D*>(d) = *reinterpret_cast<const typename Words<G>::D*>(a.scales[which] + row * G);
#pragma unroll
        for (int g = 0; g < G; g++) {
            __half2 v[4];
            q4_pairs(w[g], v);
            const __half2 dd = __half2half2(d[g]);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = __hmul2(v[j], dd);
            T* dst = reinterpret_cast<T*>(a.dst[which]) + i * a.ld[which] + head * HD + g * kQ4Group + block * 8;
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
            } else {
                const float2 f0 = __half22float2(v[0]), f1 = __half22float2(v[1]), f2 = __half22float2(v[2]), f3 = __half22float2(v[3]);
                *reinterpret_cast<float4*>(dst) = make_float4(f0.x, f0.y, f1.x, f1.y);
                *reinterpret_cast<float4*>(dst + 4) = make_float4(f2.x, f2.y, f3.x, f3.y);
            }
        }
    }
}

dim3 rows_grid(int64_t n, int kv_heads) {
    return dim3((unsigned)((kv_heads * 4 + kThreads - 1) / kThreads), (unsigned)std::min<int64_t>(n, 65535), 2);
}

int check_dims(const char* who, int32_t kv_heads, int32_t max_seq_len, int32_t head_dim) {
    if (kv_heads < 1 || kv_heads > 65536 || max_seq_len < 1) return rlb_fail(RLB_ERR_INVALID, "%s: bad kv_heads %d or max_seq_len %d", who, kv_heads, max_seq_len);
    if (max_seq_len > kMaxPositions) return rlb_fail(RLB_ERR_LIMIT, "%s: max_seq_len %d is more than %d", who, max_seq_len, kMaxPositions);
    if (head_dim != 64 && head_dim != 128) return rlb_fail(RLB_ERR_INVALID, "%s: head_dim %d is not supported (64 or 128)", who, head_dim);
    return RLB_OK;
}

// Rows of K or V given to or taken from the cache at positions start .. start + rows - 1.
int check_rows(const char* who, const rlb_cache4* c, const rlb_tensor* t, int64_t n, int32_t start) {
    if (t->ctx != c->ctx) return rlb_fail(RLB_ERR_INVALID, "%s: the rows and the cache live on different contexts", who);
    if (t->rows != n || t->cols != (int64_t)c->kv_heads * c->hd) return rlb_fail(RLB_ERR_INVALID, "%s: rows must be n x kv_heads*head_dim", who);
    if (start < 0 || start + n > c->max_seq) return rlb_fail(RLB_ERR_INVALID, "%s: positions %d..%lld are outside the cache's %d", who, start, (long long)(start + n), c->max_seq);
    return RLB_OK;
}

}  // namespace

extern "C" {

int rlb_cache4_create(rlb_ctx* ctx, int32_t kv_heads, int32_t max_seq_len, int32_t head_dim, rlb_cache4** out) {
    if (!ctx || !out) return rlb_fail(RLB_ERR_INVALID, "rlb_cache4_create: null pointer");
    *out = nullptr;
    RLB_TRY(check_dims("rlb_cache4_create", kv_heads, max_seq_len, head_dim));
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    DeviceScope dev(ctx->device);
    RLB_CUDA(dev.err);
    if (ctx_capturing(ctx)) return rlb_fail(RLB_ERR_STATE, "rlb_cache4_create allocates: it cannot be captured into a graph");
    OutsideCapture now;
    const size_t rows = (size_t)kv_heads * max_seq_len;
    const size_t codes = (rows * (head_dim / 2) + 255) & ~(size_t)255, scales = (rows * (head_dim / kQ4Group) * 2 + 255) & ~(size_t)255;
    rlb_cache4* c = new (std::nothrow) rlb_cache4();
    if (!c) return rlb_fail(RLB_ERR_OOM, "rlb_cache4_create: out of host memory");
    cudaError_t e = cudaMalloc(&c->owned, 2 * (codes + scales));
    if (e != cudaSuccess) {
        delete c;
        return rlb_fail(RLB_ERR_OOM, "rlb_cache4_create: cudaMalloc(%zu): %s", 2 * (codes + scales), cudaGetErrorString(e));
    }
    e = cudaMemsetAsync(c->owned, 0, 2 * (codes + scales), ctx->stream);  // scale 0: every value is zero
    if (e != cudaSuccess) {
        cudaFree(c->owned);
        delete c;
        return rlb_fail(RLB_ERR_CUDA, "rlb_cache4_create: %s", cudaGetErrorString(e));
    }
    uint8_t* p = (uint8_t*)c->owned;
    c->codes[0] = p; c->codes[1] = p + codes;
    c->scales[0] = (__half*)(p + 2 * codes); c->scales[1] = (__half*)(p + 2 * codes + scales);
    c->ctx = ctx; c->device = ctx->device; c->kv_heads = kv_heads; c->max_seq = max_seq_len; c->hd = head_dim;
    *out = c;
    return RLB_OK;
}

int rlb_cache4_wrap(rlb_ctx* ctx, void* k_codes, void* k_scales, void* v_codes, void* v_scales, int32_t kv_heads, int32_t max_seq_len,
                    int32_t head_dim, rlb_cache4** out) {
    if (!ctx || !out) return rlb_fail(RLB_ERR_INVALID, "rlb_cache4_wrap: null pointer");
    *out = nullptr;
    RLB_TRY(check_dims("rlb_cache4_wrap", kv_heads, max_seq_len, head_dim));
    const size_t rows = (size_t)kv_heads * max_seq_len;
    const struct { const void* p; size_t bytes; } parts[] = {{k_codes, rows * (head_dim / 2)}, {k_scales, rows * (head_dim / kQ4Group) * 2},
                                                             {v_codes, rows * (head_dim / 2)}, {v_scales, rows * (head_dim / kQ4Group) * 2}};
    for (const auto& part : parts) {
        if (!part.p || ((uintptr_t)part.p & 15)) return rlb_fail(RLB_ERR_INVALID, "rlb_cache4_wrap: the four arrays must be 16-byte aligned");
        RLB_TRY(check_device_memory(ctx, part.p, "rlb_cache4_wrap"));
        RLB_TRY(check_device_memory(ctx, (const char*)part.p + part.bytes - 1, "rlb_cache4_wrap: the last element"));
    }
    rlb_cache4* c = new (std::nothrow) rlb_cache4();
    if (!c) return rlb_fail(RLB_ERR_OOM, "rlb_cache4_wrap: out of host memory");
    c->codes[0] = (uint8_t*)k_codes; c->codes[1] = (uint8_t*)v_codes;
    c->scales[0] = (__half*)k_scales; c->scales[1] = (__half*)v_scales;
    c->ctx = ctx; c->device = ctx->device; c->kv_heads = kv_heads; c->max_seq = max_seq_len; c->hd = head_dim;
    *out = c;
    return RLB_OK;
}

int rlb_cache4_free(rlb_cache4* c) {
    if (!c) return RLB_OK;
    if (c->owned) {
        DeviceScope dev(c->device);
        OutsideCapture now;
        cudaFree(c->owned);  // waits for the device
    }
    delete c;
    return RLB_OK;
}

int rlb_cache4_append(rlb_cache4* c, const rlb_tensor* k, const rlb_tensor* v, int32_t start_pos) {
    if (!c || !k || !v) return rlb_fail(RLB_ERR_INVALID, "rlb_cache4_append: null pointer");
    RLB_TRY(check_rows("rlb_cache4_append", c, k, k->rows, start_pos));
    RLB_TRY(check_rows("rlb_cache4_append", c, v, k->rows, start_pos));
    if (k->dtype != v->dtype) return rlb_fail(RLB_ERR_INVALID, "rlb_cache4_append: K and V rows must have one dtype");
    if (k->rows == 0) return RLB_OK;
    rlb_ctx* ctx = c->ctx;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    DeviceScope dev(ctx->device);
    RLB_CUDA(dev.err);
    AppendArgs a = {};
    a.src[0] = k->d; a.src[1] = v->d; a.ld[0] = k->cap; a.ld[1] = v->cap;
    for (int w = 0; w < 2; w++) { a.codes[w] = c->codes[w]; a.scales[w] = c->scales[w]; }
    a.kv_heads = c->kv_heads; a.max_seq = c->max_seq; a.start = start_pos;
    a.n = (int)k->rows;
    const dim3 grid = rows_grid(k->rows, 2 * c->kv_heads);
    if (k->dtype == RLB_F16) {
        if (c->hd == 128) append4_kernel<__half, 128, false><<<grid, kThreads, 0, ctx->stream>>>(a);
        else append4_kernel<__half, 64, false><<<grid, kThreads, 0, ctx->stream>>>(a);
    } else {
        if (c->hd == 128) append4_kernel<float, 128, false><<<grid, kThreads, 0, ctx->stream>>>(a);
        else append4_kernel<float, 64, false><<<grid, kThreads, 0, ctx->stream>>>(a);
    }
    RLB_LAUNCH_CHECK();
    count_launch(ctx);
    return RLB_OK;
}

int rlb_cache4_norm_rope_append(rlb_cache4* c, rlb_tensor* q_out, const rlb_tensor* q, const rlb_tensor* k, const rlb_tensor* v,
                                const rlb_tensor* q_gain, const rlb_tensor* k_gain, float eps, const rlb_tensor* rope, int32_t heads, int32_t start_pos) {
    const char* who = "rlb_cache4_norm_rope_append";
    if (!c || !q_out || !q || !k || !v || !rope) return rlb_fail(RLB_ERR_INVALID, "%s: null pointer", who);
    RLB_TRY(check_rows(who, c, k, q->rows, start_pos));
    RLB_TRY(check_rows(who, c, v, q->rows, start_pos));
    const int64_t n = q->rows, hd = c->hd;
    if (q->ctx != c->ctx || q_out->ctx != c->ctx || rope->ctx != c->ctx) return rlb_fail(RLB_ERR_INVALID, "%s: the rows and the cache live on different contexts", who);
    for (const rlb_tensor* g : {q_gain, k_gain})
        if (g && (g->ctx != c->ctx || g->dtype != RLB_F32 || g->rows != 1 || g->cols != hd)) return rlb_fail(RLB_ERR_INVALID, "%s: a gain must be 1 x head_dim f32", who);
    if (heads < 1 || heads > 65536) return rlb_fail(RLB_ERR_INVALID, "%s: bad heads %d", who, heads);
    if (q->dtype != RLB_F32 || q->cols != heads * hd || q_out->dtype != RLB_F32 || q_out->rows != n || q_out->cols != q->cols)
        return rlb_fail(RLB_ERR_INVALID, "%s: q and q_out must be n x heads*head_dim f32", who);
    if (k->dtype != RLB_F32 || v->dtype != RLB_F32) return rlb_fail(RLB_ERR_INVALID, "%s: k and v must be f32", who);
    if (rope->dtype != RLB_F32 || rope->cols != hd || rope->rows < start_pos + n)
        return rlb_fail(RLB_ERR_INVALID, "%s: the rope table must be f32, head_dim wide and cover position %lld", who, (long long)(start_pos + n - 1));
    if (!(eps >= 0.f)) return rlb_fail(RLB_ERR_INVALID, "%s: eps must not be negative", who);
    if (n == 0) return RLB_OK;
    rlb_ctx* ctx = c->ctx;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    DeviceScope dev(ctx->device);
    RLB_CUDA(dev.err);
    AppendArgs a = {};
    a.src[0] = k->d; a.src[1] = v->d; a.src[2] = q->d; a.ld[0] = k->cap; a.ld[1] = v->cap; a.ld[2] = q->cap;
    for (int w = 0; w < 2; w++) { a.codes[w] = c->codes[w]; a.scales[w] = c->scales[w]; }
    a.kv_heads = c->kv_heads; a.max_seq = c->max_seq; a.start = start_pos; a.n = (int)n;
    a.q_out = (float*)q_out->d; a.qo_ld = q_out->cap;
    a.gain[0] = k_gain ? (const float*)k_gain->d : nullptr; a.gain[2] = q_gain ? (const float*)q_gain->d : nullptr;
    a.table = (const float*)rope->d; a.table_ld = rope->cap; a.eps = eps; a.heads = heads;
    dim3 grid = rows_grid(n, 2 * std::max(c->kv_heads, (int)heads));
    grid.z = 3;
    if (hd == 128) append4_kernel<float, 128, true><<<grid, kThreads, 0, ctx->stream>>>(a);
    else append4_kernel<float, 64, true><<<grid, kThreads, 0, ctx->stream>>>(a);
    RLB_LAUNCH_CHECK();
    count_launch(ctx);
    return tensor_mark_ready(q_out);
}

int rlb_cache4_read(rlb_cache4* c, rlb_tensor* k_out, rlb_tensor* v_out, int32_t start_pos) {
    if (!c || (!k_out && !v_out)) return rlb_fail(RLB_ERR_INVALID, "rlb_cache4_read: null pointer");
    const rlb_tensor* any = k_out ? k_out : v_out;
    if (k_out) RLB_TRY(check_rows("rlb_cache4_read", c, k_out, any->rows, start_pos));
    if (v_out) RLB_TRY(check_rows("rlb_cache4_read", c, v_out, any->rows, start_pos));
    if (k_out && v_out && k_out->dtype != v_out->dtype) return rlb_fail(RLB_ERR_INVALID, "rlb_cache4_read: K and V rows must have one dtype");
    if (any->rows == 0) return RLB_OK;
    rlb_ctx* ctx = c->ctx;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    DeviceScope dev(ctx->device);
    RLB_CUDA(dev.err);
    ReadArgs a;
    a.dst[0] = k_out ? k_out->d : nullptr; a.dst[1] = v_out ? v_out->d : nullptr;
    a.ld[0] = k_out ? k_out->cap : 0; a.ld[1] = v_out ? v_out->cap : 0;
    for (int w = 0; w < 2; w++) { a.codes[w] = c->codes[w]; a.scales[w] = c->scales[w]; }
    a.kv_heads = c->kv_heads; a.max_seq = c->max_seq; a.start = start_pos;
    a.n = (int)any->rows;
    const dim3 grid = rows_grid(any->rows, c->kv_heads);
    if (any->dtype == RLB_F16) {
        if (c->hd == 128) read4_kernel<__half, 128><<<grid, kThreads, 0, ctx->stream>>>(a);
        else read4_kernel<__half, 64><<<grid, kThreads, 0, ctx->stream>>>(a);
    } else {
        if (c->hd == 128) read4_kernel<float, 128><<<grid, kThreads, 0, ctx->stream>>>(a);
        else read4_kernel<float, 64><<<grid, kThreads, 0, ctx->stream>>>(a);
    }
    RLB_LAUNCH_CHECK();
    count_launch(ctx);
    if (k_out) RLB_TRY(tensor_mark_ready(k_out));
    if (v_out) RLB_TRY(tensor_mark_ready(v_out));
    return RLB_OK;
}

}  // extern "C"
