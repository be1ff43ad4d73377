// Attention for long contexts: a sliding window with first tokens that stay visible, K/V heads shared by several query
// heads, and caches in f32, f16 or 4 bits (cache4.h). The per-head part of Attention::forward (src/transformer.rs:727-781)
// with the visible set narrowed: query row i, at position p = start + i, sees
//     t <= p  and  (t > p - window  or  t < sinks),
// out_i = sum_t exp(s_t) v_t / sum_t exp(s_t), s_t = q . k_t / sqrt(head_dim), in f32 with the running maximum taken out.
// A row that sees nothing (window 0 and no first tokens) is zero. Cache rows that a query row does not see never reach its
// result, whatever they hold.
//
// The union of what the positions p0..p1 see is two runs, [0, S) and [L, p1 + 1) with L = max(0, p0 + 1 - window) and
// S = min(sinks, L); kernels walk it as one virtual index v -> v < S ? v : v - S + L.
#include "attention_long.h"

#include <algorithm>

using namespace attn_long;

namespace {

// One query row over an f32 cache: a CTA of eight warps, a warp per position, lanes over head_dim; grid (rows, splits). A row reads what it sees for
// itself, so the bound is the caches' reading for one row and L2 for several (8 rows after 10000 positions, 32 heads: 306 us, 8.6 TB/s from L2);
// 77 rows of 8 heads on 4, window 100, are 8.8 us, half of them the call. Four rows of a K/V head to a CTA, each position fetched once for them, are no
// faster (that case 15.6, 16 rows after 4000 positions 186 against 117; only 64 heads on 8 gain, 208 to 194), nor are two or four positions of a warp at
// a time: more registers, fewer warps.
template <int HD>
__global__ void __launch_bounds__(256) attn_long_row_kernel(const AttnLongArgs a) {
    constexpr int N = HD / 32;
    __shared__ float w_o[8][HD], w_m[8], w_l[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x;
    const int i = (int)(r / a.heads), head = (int)(r % a.heads), p = a.start + i;
    const Run run = visible_run(a, p, p);
    const int chunk = (run.len + a.n_split - 1) / a.n_split;
    const int v0 = min(run.len, (int)blockIdx.y * chunk), v1 = min(run.len, v0 + chunk);
    const int64_t base = (int64_t)(head / a.group) * a.max_seq;
    PlainRow<CACHE_F32, HD> one(a, i, head, lane);
    for (int v = v0 + warp; v < v1; v += 8) one.see(a, base + run.at(v), lane);
    if (lane == 0) { w_m[warp] = one.m; w_l[warp] = one.l; }
#pragma unroll
    for (int e = 0; e < N; e++) w_o[warp][lane * N + e] = one.o[e];
    __syncthreads();
    if (threadIdx.x >= HD) return;
    float M = -FLT_MAX, L = 0.f, O = 0.f;
    for (int w = 0; w < 8; w++) M = fmaxf(M, w_m[w]);
    for (int w = 0; w < 8; w++) {
        const float f = exp2f(w_m[w] - M);
        L = fmaf(w_l[w], f, L);
        O = fmaf(w_o[w][threadIdx.x], f, O);
    }
    if (a.n_split > 1) {
        const int64_t rec = r * a.n_split + blockIdx.y;
        a.rec_o[rec * HD + threadIdx.x] = O;
        if (threadIdx.x == 0) a.rec_ml[rec] = make_float2(M, L);
    } else {
        store_out(reinterpret_cast<float*>(a.out) + i * a.out_ld + head * HD + threadIdx.x, run.len > 0 ? O / L : 0.f);
    }
}

// Joins the splits of a row. W warps share a row (each takes every W-th split), a lane has HD / 32 columns; a CTA of eight warps. W = 1 for up
// to eight splits: 20480 rows of three splits take 29 us with eight warps to a row, five of them idle.
template <typename OT, int HD, int W>
__global__ void __launch_bounds__(256) attn_long_merge_kernel(const __grid_constant__ AttnLongArgs a) {
    constexpr int N = HD / 32;
    __shared__ float o_s[W == 1 ? 1 : 8][HD], m_s[8], l_s[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = W == 1 ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;
    rlb_pdl_wait();   // launched while the kernel that writes the records drains
    if (r >= (int64_t)a.n * a.heads) return;
    const int i = (int)(r / a.heads), head = (int)(r % a.heads), p = a.start + i;
    const float2* ml = a.rec_ml + r * a.n_split;
    const float* rec = a.rec_o + r * a.n_split * HD + lane * N;
    float m = -FLT_MAX, l = 0.f, o[N] = {};
#pragma unroll 4
    for (int s = W == 1 ? 0 : warp; s < a.n_split; s += W) {
        const float2 x = ml[s];
        float y[N];
        if constexpr (N == 4) *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(rec + (int64_t)s * HD);
        else *reinterpret_cast<float2*>(y) = *reinterpret_cast<const float2*>(rec + (int64_t)s * HD);
        const float m_new = fmaxf(m, x.x), f = exp2f(m - m_new), g = exp2f(x.x - m_new);
        l = l * f + x.y * g;
#pragma unroll
        for (int e = 0; e < N; e++) o[e] = o[e] * f + y[e] * g;
        m = m_new;
    }
    const bool sees = visible_run(a, p, p).len > 0;
    OT* out = reinterpret_cast<OT*>(a.out) + i * a.out_ld + head * HD;
    if constexpr (W == 1) {
        const float inv = 1.0f / l;
#pragma unroll
        for (int e = 0; e < N; e++) o[e] = sees ? o[e] * inv : 0.f;
        if constexpr (sizeof(OT) == 4) {
#pragma unroll
            for (int e = 0; e < N; e += 2) *reinterpret_cast<float2*>(out + lane * N + e) = make_float2(o[e], o[e + 1]);
        } else {
#pragma unroll
            for (int e = 0; e < N; e += 2) *reinterpret_cast<__half2*>(out + lane * N + e) = mean_f16(o[e], o[e + 1]);
        }
        return;
    }
    if (lane == 0) { m_s[warp] = m; l_s[warp] = l; }
#pragma unroll
    for (int e = 0; e < N; e++) o_s[W == 1 ? 0 : warp][lane * N + e] = o[e];
    __syncthreads();
    if (threadIdx.x >= HD) return;
    float M = -FLT_MAX, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) M = fmaxf(M, m_s[w]);
#pragma unroll
    for (int w = 0; w < 8; w++) {
        const float f = exp2f(m_s[w] - M);
        L = fmaf(l_s[w], f, L);
        O = fmaf(o_s[W == 1 ? 0 : w][threadIdx.x], f, O);
    }
    store_out(out + threadIdx.x, sees ? O / L : 0.f);
}

template <typename OT, int HD>
int launch_merge(rlb_ctx* ctx, const AttnLongArgs& a) {
    cudaLaunchConfig_t lc = {};
    const int64_t rows = (int64_t)a.n * a.heads;
    const bool single = a.n_split <= 8;
    lc.gridDim = dim3((unsigned)(single ? (rows + 7) / 8 : rows));
    lc.blockDim = dim3(256);
    lc.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    if (single) RLB_CUDA(cudaLaunchKernelEx(&lc, attn_long_merge_kernel<OT, HD, 1>, a));
    else RLB_CUDA(cudaLaunchKernelEx(&lc, attn_long_merge_kernel<OT, HD, 8>, a));
    count_launch(ctx);
    return RLB_OK;
}

template <int HD>
int launch_rows(rlb_ctx* ctx, const AttnLongArgs& a) {
    attn_long_row_kernel<HD><<<dim3((unsigned)(a.n * a.heads), a.n_split), 256, 0, ctx->stream>>>(a);
    RLB_LAUNCH_CHECK();
    count_launch(ctx);
    return RLB_OK;
}
int rows_splits(rlb_ctx* ctx, const AttnLongArgs& a) {
    // Eight CTAs an SM, and at least 64 positions to a split, but 128 to the only one: the second kernel costs as much. (77 rows of 8 heads, window
    // 100: one split 9.4 us, two 11.4; 16 rows of 8 heads, window 200: two 10.4, four 8.6.)
    if (ctx->attn_long_splits) return ctx->attn_long_splits;
    const int64_t rows = (int64_t)a.n * a.heads, most = std::min<int64_t>((int64_t)a.sinks + a.window, (int64_t)a.start + a.n);
    if (most <= 128) return 1;
    const int64_t splits = std::min<int64_t>((8 * ctx->sm_count + rows - 1) / rows, (most + 63) / 64);
    return (int)std::max<int64_t>(1, std::min<int64_t>(splits, 256));
}

// What both entry points require of q, out and the visible set.
int check(const char* who, const rlb_tensor* out, const rlb_tensor* q, rlb_dtype out_dtype, int32_t heads, int32_t kv_heads, int32_t max_seq,
          int64_t hd, int32_t start, int32_t window, int32_t sinks) {
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0) return rlb_fail(RLB_ERR_INVALID, "%s: heads %d is not a multiple of kv_heads %d", who, heads, kv_heads);
    if (hd != 64 && hd != 128) return rlb_fail(RLB_ERR_INVALID, "%s: head_dim %lld is not supported (64 or 128)", who, (long long)hd);
    if (max_seq < 1 || start < 0 || start + q->rows > max_seq)
        return rlb_fail(RLB_ERR_INVALID, "%s: bad max_seq_len %d, start_pos %d or %lld rows", who, max_seq, start, (long long)q->rows);
    if (max_seq > kMaxPositions) return rlb_fail(RLB_ERR_LIMIT, "%s: max_seq_len %d is more than %d", who, max_seq, kMaxPositions);
    if (window < 0 || sinks < 0) return rlb_fail(RLB_ERR_INVALID, "%s: window %d and sinks %d must not be negative", who, window, sinks);
    if (q->dtype != RLB_F32 || q->cols != heads * hd) return rlb_fail(RLB_ERR_INVALID, "%s: q must be n x heads*head_dim f32", who);
    if (q->cols > kMaxColumns) return rlb_fail(RLB_ERR_LIMIT, "%s: rows of %lld columns are more than %lld", who, (long long)q->cols, (long long)kMaxColumns);
    if (out->dtype != out_dtype || out->rows != q->rows || out->cols != q->cols)
        return rlb_fail(RLB_ERR_INVALID, "%s: out must be n x heads*head_dim in %s", who, out_dtype == RLB_F16 ? "f16" : "f32");
    if (out->d == q->d && q->rows > 0) return rlb_fail(RLB_ERR_INVALID, "%s: out and q are one tensor", who);
    if (q->rows * heads > 0x7fffffffll) return rlb_fail(RLB_ERR_LIMIT, "%s: %lld rows of %d heads are more than one launch takes", who, (long long)q->rows, heads);
    return RLB_OK;
}

int run(CacheKind kind, AttnLongArgs& a, rlb_tensor* out, const rlb_tensor* q, int32_t heads, int32_t kv_heads, int32_t max_seq, int64_t hd,
        int32_t start, int32_t window, int32_t sinks) {
    if (q->rows == 0) return RLB_OK;
    rlb_ctx* ctx = out->ctx;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    DeviceScope dev(ctx->device);
    RLB_CUDA(dev.err);
    a.q = (const float*)q->d; a.q_ld = q->cap; a.out = out->d; a.out_ld = out->cap;
    a.n = (int)q->rows; a.heads = heads; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.hd = (int)hd; a.max_seq = max_seq;
    a.start = start; a.window = window; a.sinks = sinks;
    RLB_TRY(launch_attn_long(ctx, kind, a));
    return tensor_mark_ready(out);
}

}  // namespace

int launch_attn_long(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& given) {
    AttnLongArgs a = given;
    const bool f32 = kind == CACHE_F32;
    AttnSplit split;
    bool tiles, few = false;
    if (f32) {
        // Tiles of 64 rows of a K/V head, 15 us (head_dim 128) for 64 positions of two of them an SM, or row by row, 0.12 us for 1000 scores. (32 heads,
        // 10000 positions: 8 rows 306 us row by row, 16 rows 285 in tiles; 8 heads of 64 on 4 K/V heads, 77 rows, window 100: 10 row by row, 20 in tiles.)
        const int t = attn_long_f32_splits(ctx, a), r = rows_splits(ctx, a);
        const int64_t seen = std::min<int64_t>((int64_t)a.window + a.sinks, (int64_t)a.start + a.n);
        const double row_us = 5 + 0.12e-3 * (double)a.n * a.heads * (double)seen * (a.hd == 128 ? 1 : 0.7);
        tiles = ctx->attn_long ? ctx->attn_long == 2 : attn_long_f32_us(ctx, a, t) < row_us;
        split.n = tiles ? t : r;
        split.records = split.n > 1;
    } else {
        // The kernel for few rows reads the cache once for every eight of them, the one for many rows has tiles of 128 (256 in 4 bits) that cost
        // the same however many of their rows there are. Each says what it expects to take, from what was measured; e.g. 32
        // heads, 8000 positions, us with few / tiles: f16 8 rows 30 / 33, 16 rows 47 / 34, 64 rows 161 / 39; 4 bits 8 rows 20 / 43, 24 rows 60 / 44, 64
        // rows 103 / 45; 300 positions: f16 32 rows 8 / 12, 64 rows 14 / 12; 4 bits 64 rows 10 / 15, 128 rows 18 / 16. Not covered: prompts with windows
        // of up to 16 positions (4 bits, narrow heads: up to 64). A round of CTAs of the kernel for few rows costs about 4 us (4 bits 5.5) however little it
        // reads, which its estimate leaves out: 1792 rows of 64 heads, window 4, take 378 us where tiles take 47 (4 bits 265 and 71). With wider windows the
        // choice was right in all of the shapes measured but one: 512 rows of 8 heads of 64, window 256, 15.9 and 12.1.
        const AttnSplit s = attn_long_few_splits(ctx, kind, a);
        const int t = attn_long_tc_splits(ctx, kind, a);
        few = ctx->attn_long ? ctx->attn_long == 1 : attn_long_few_us(ctx, kind, a, s) <= attn_long_tc_us(ctx, kind, a, t);
        tiles = !few;
        split = few ? s : AttnSplit{t, t > 1};
    }
    const int64_t rows = (int64_t)a.n * a.heads;
    OpWorkspace ws;
    if (split.records) {
        const size_t recs = (size_t)rows * split.n;
        const int got = ws.get(ctx, recs * (a.hd * sizeof(float) + sizeof(float2)));
        if (got == RLB_OK) {
            a.rec_o = (float*)ws.p;
            a.rec_ml = (float2*)(a.rec_o + recs * a.hd);
        } else if (got == RLB_ERR_OOM && !ctx_capturing(ctx)) {
            split = {1, false};   // no memory for records: slower without them
        } else {
            return got;
        }
    }
    a.n_split = split.n;
    if (few) RLB_TRY(launch_attn_long_few(ctx, kind, a));
    else if (!f32) RLB_TRY(launch_attn_long_tc(ctx, kind, a));
    else if (tiles) RLB_TRY(launch_attn_long_f32(ctx, a));
    else RLB_TRY(a.hd == 128 ? launch_rows<128>(ctx, a) : launch_rows<64>(ctx, a));
    if (split.records) {
        if (f32) RLB_TRY(a.hd == 128 ? (launch_merge<float, 128>(ctx, a)) : (launch_merge<float, 64>(ctx, a)));
        else RLB_TRY(a.hd == 128 ? (launch_merge<__half, 128>(ctx, a)) : (launch_merge<__half, 64>(ctx, a)));
    }
    return RLB_OK;
}

extern "C" int rlb_attention_window(rlb_tensor* out, const rlb_tensor* q, const rlb_tensor* kcache, const rlb_tensor* vcache, int32_t heads,
                                    int32_t kv_heads, int32_t max_seq_len, int32_t start_pos, int32_t window, int32_t sinks) {
    RLB_TRY(same_ctx(out, q));
    RLB_TRY(same_ctx(out, kcache));
    RLB_TRY(same_ctx(out, vcache));
    const int64_t hd = kcache->cols;
    RLB_TRY(check("attention_window", out, q, kcache->dtype, heads, kv_heads, max_seq_len, hd, start_pos, window, sinks));
    if (kcache->cap != hd || vcache->cap != hd || vcache->cols != hd || kcache->rows != (int64_t)kv_heads * max_seq_len ||
        vcache->rows != kcache->rows || kcache->dtype != vcache->dtype)
        return rlb_fail(RLB_ERR_INVALID, "attention_window: caches must be (kv_heads*max_seq_len) x head_dim without row padding");
    AttnLongArgs a;
    a.k = kcache->d; a.v = vcache->d;
    return run(kcache->dtype == RLB_F16 ? CACHE_F16 : CACHE_F32, a, out, q, heads, kv_heads, max_seq_len, hd, start_pos, window, sinks);
}

extern "C" int rlb_cache4_attention(rlb_cache4* c, rlb_tensor* out, const rlb_tensor* q, int32_t heads, int32_t start_pos, int32_t window, int32_t sinks) {
    if (!c) return rlb_fail(RLB_ERR_INVALID, "rlb_cache4_attention: null cache");
    RLB_TRY(same_ctx(out, q));
    if (out->ctx != c->ctx) return rlb_fail(RLB_ERR_INVALID, "rlb_cache4_attention: the rows and the cache live on different contexts");
    RLB_TRY(check("rlb_cache4_attention", out, q, RLB_F16, heads, c->kv_heads, c->max_seq, c->hd, start_pos, window, sinks));
    AttnLongArgs a;
    a.k = c->codes[0]; a.v = c->codes[1]; a.k_scale = c->scales[0]; a.v_scale = c->scales[1];
    return run(CACHE_Q4, a, out, q, heads, c->kv_heads, c->max_seq, c->hd, start_pos, window, sinks);
}
