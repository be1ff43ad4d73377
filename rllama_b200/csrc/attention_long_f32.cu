// Long-context attention of many query rows over f32 caches: attention_long.cu says what is computed. f32 products and sums throughout (no
// tensor-core format keeps 24 bits), so the FMA pipes are the bound and registers are tiled for them: a CTA takes 64 rows (row = i * group + g
// of a K/V head, as in attention_long_tc.cu) and walks the positions that some of them see 64 at a time; a thread computes 4 x 4 scores,
// then 4 x HD / 16 columns of the result, from operands that lie in shared memory in rows padded by 16 bytes (8 and 12 vector loads for 64 and
// 128 FMAs). The weights take the place of the K tile. Two CTAs share an SM: one's loads fall into the other's arithmetic.
// 400 rows after 8000 positions, 40 heads: 1.97 ms, 34 TFLOP/s (of about 75 that the FMA pipes have).
// A zero weight times an infinite or NaN value is a NaN here too; rows with a NaN that their sum does not have are computed again, one warp to a row.
#include <algorithm>

#include "attention_long.h"

using namespace attn_long;

namespace {

constexpr int QT = 64, TK = 64, kThreads = 256;

template <int HD> struct Shape {
    static constexpr int LD = HD + 4, LP = TK + 4;
    static constexpr int KF = TK * LD > QT * LP ? TK * LD : QT * LP;   // K tile, then weights
    static constexpr size_t SMEM = sizeof(float) * (size_t)(QT * LD + KF + TK * LD);
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 2) attn_long_f32_kernel(const __grid_constant__ AttnLongArgs a) {
    constexpr int LD = Shape<HD>::LD, LP = Shape<HD>::LP, NC = HD / 64;   // NC: float4 column groups of a thread's result
    extern __shared__ __align__(16) float sm[];
    float *q_s = sm, *k_s = q_s + QT * LD, *v_s = k_s + Shape<HD>::KF, *p_s = k_s;
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
    const int kvh = blockIdx.x % a.kv_heads, n_rows = a.n * a.group;
    const int row0 = ((n_rows + QT - 1) / QT - 1 - (int)blockIdx.x / a.kv_heads) * QT, row_last = min(n_rows, row0 + QT) - 1;
    const Run run = visible_run(a, a.start + row0 / a.group, a.start + row_last / a.group);
    int chunk = (run.len + a.n_split - 1) / a.n_split;
    chunk = (chunk + TK - 1) / TK * TK;
    const int v0 = min(run.len, (int)blockIdx.y * chunk), v1 = min(run.len, v0 + chunk);
    const float* k = reinterpret_cast<const float*>(a.k) + (int64_t)kvh * a.max_seq * HD;
    const float* v = reinterpret_cast<const float*>(a.v) + (int64_t)kvh * a.max_seq * HD;
    const float c2 = rsqrtf((float)HD) * 1.4426950408889634f;
    for (int e = tid; e < QT * (HD / 4); e += kThreads) {
        const int y = e / (HD / 4), c = e % (HD / 4) * 4, row = row0 + y;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row <= row_last) x = *reinterpret_cast<const float4*>(a.q + (int64_t)(row / a.group) * a.q_ld + (int64_t)(kvh * a.group + row % a.group) * HD + c);
        *reinterpret_cast<float4*>(q_s + y * LD + c) = make_float4(x.x * c2, x.y * c2, x.z * c2, x.w * c2);
    }
    int p[4], low[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        p[i] = a.start + min(row0 + ty * 4 + i, row_last) / a.group;
        low[i] = window_low(a, p[i]);
    }
    float m[4], l[4], o[4][NC][4] = {};
#pragma unroll
    for (int i = 0; i < 4; i++) { m[i] = -FLT_MAX; l[i] = 0.f; }

    for (int w0 = v0; w0 < v1; w0 += TK) {
        __syncthreads();   // the tiles before are used, q_s is there
        for (int half = 0; half < 2; half++) {
            const float* src = half ? v : k;
            float* dst = half ? v_s : k_s;
            for (int e = tid; e < TK * (HD / 4); e += kThreads) {
                const int y = e / (HD / 4), c = e % (HD / 4) * 4, w = w0 + y;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + y * LD + c)),
                             "l"(src + (int64_t)run.at(min(w, v1 - 1)) * HD + c), "r"(w < v1 ? 16 : 0)   // (zeros behind the end)
                             : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
        float s[4][4] = {};
#pragma unroll 4
        for (int d = 0; d < HD; d += 4) {
            float4 qv[4], kv[4];
#pragma unroll
            for (int i = 0; i < 4; i++) qv[i] = *reinterpret_cast<const float4*>(q_s + (ty * 4 + i) * LD + d);
#pragma unroll
            for (int j = 0; j < 4; j++) kv[j] = *reinterpret_cast<const float4*>(k_s + (tx + 16 * j) * LD + d);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    s[i][j] = fmaf(qv[i].x, kv[j].x, s[i][j]);
                    s[i][j] = fmaf(qv[i].y, kv[j].y, s[i][j]);
                    s[i][j] = fmaf(qv[i].z, kv[j].z, s[i][j]);
                    s[i][j] = fmaf(qv[i].w, kv[j].w, s[i][j]);
                }
        }
        __syncthreads();   // K is used: the weights take its place
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int w = w0 + tx + 16 * j, t = run.at(w);
                if (!(w < v1 && t <= p[i] && (t >= low[i] || t < a.sinks))) s[i][j] = -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float m_new = fmaxf(m[i], top), scale = exp2f(m[i] - m_new);
            m[i] = m_new;
            l[i] *= scale;
#pragma unroll
            for (int g = 0; g < NC; g++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][g][e] *= scale;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float w = exp2f(s[i][j] - m_new);
                l[i] += w;
                p_s[(ty * 4 + i) * LP + tx + 16 * j] = w;
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
#pragma unroll 2
        for (int t = 0; t < TK; t += 4) {
            float4 pv[4];
#pragma unroll
            for (int i = 0; i < 4; i++) pv[i] = *reinterpret_cast<const float4*>(p_s + (ty * 4 + i) * LP + t);
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int g = 0; g < NC; g++) {
                    const float4 vv = *reinterpret_cast<const float4*>(v_s + (t + x) * LD + g * 64 + tx * 4);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float w = x == 0 ? pv[i].x : x == 1 ? pv[i].y : x == 2 ? pv[i].z : pv[i].w;
                        o[i][g][0] = fmaf(w, vv.x, o[i][g][0]);
                        o[i][g][1] = fmaf(w, vv.y, o[i][g][1]);
                        o[i][g][2] = fmaf(w, vv.z, o[i][g][2]);
                        o[i][g][3] = fmaf(w, vv.w, o[i][g][3]);
                    }
                }
        }
    }
    __shared__ uint32_t bad[2];
    if (tid < 2) bad[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float sum = l[i];
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const int y = ty * 4 + i, row = row0 + y;
        if (row > row_last) continue;
        const int ii = row / a.group, head = kvh * a.group + row % a.group;
        const bool sees = visible_run(a, p[i], p[i]).len > 0;
        const float inv = a.n_split > 1 ? 1.f : sees ? 1.0f / sum : 0.f;
        const int64_t rec = ((int64_t)ii * a.heads + head) * a.n_split + blockIdx.y;
        float* dst = a.n_split > 1 ? a.rec_o + rec * HD : reinterpret_cast<float*>(a.out) + ii * a.out_ld + head * HD;
        float o_top = 0.f;
#pragma unroll
        for (int g = 0; g < NC; g++) {
            float4 x;
            x.x = o[i][g][0] * inv; x.y = o[i][g][1] * inv; x.z = o[i][g][2] * inv; x.w = o[i][g][3] * inv;
#pragma unroll
            for (int e = 0; e < 4; e++) max_abs_nan(o_top, o[i][g][e]);
            *reinterpret_cast<float4*>(dst + g * 64 + tx * 4) = a.n_split > 1 || sees ? x : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (a.n_split > 1 && tx == 0) a.rec_ml[rec] = make_float2(m[i], sum);
        if (sees && row_is_suspect(sum, o_top, 0.f)) atomicOr(&bad[y >> 5], 1u << (y & 31));
    }
    __syncthreads();
    // rows next to infinite or NaN cache contents that they do not see, again from what they see alone, a warp to a row
    constexpr int N = HD / 32;
    const int lane = tid & 31, warp = tid >> 5;
    for (int y = warp; y < QT; y += kThreads / 32) {
        if (!((bad[y >> 5] >> (y & 31)) & 1)) continue;
        const int row = row0 + y, ii = row / a.group, head = kvh * a.group + row % a.group, pp = a.start + ii;
        PlainRow<CACHE_F32, HD> one(a, ii, head, lane);
        for (int w = v0; w < v1; w++) {
            const int t = run.at(w);
            if (visible(a, pp, t)) one.see(a, (int64_t)kvh * a.max_seq + t, lane);
        }
        const int64_t rec = ((int64_t)ii * a.heads + head) * a.n_split + blockIdx.y;
        float* dst = a.n_split > 1 ? a.rec_o + rec * HD : reinterpret_cast<float*>(a.out) + ii * a.out_ld + head * HD;
#pragma unroll
        for (int e = 0; e < N; e++) dst[lane * N + e] = a.n_split > 1 ? one.o[e] : one.o[e] / one.l;
        if (a.n_split > 1 && lane == 0) a.rec_ml[rec] = make_float2(one.m, one.l);
    }
}

template <int HD>
int launch(rlb_ctx* ctx, const AttnLongArgs& a) {
    static std::atomic<uint64_t> set{0};
    if (!attr_done(set, ctx->device)) {
        RLB_CUDA(cudaFuncSetAttribute(attn_long_f32_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<HD>::SMEM));
        attr_mark(set, ctx->device);
    }
    const int blocks = (a.n * a.group + QT - 1) / QT;
    attn_long_f32_kernel<HD><<<dim3((unsigned)(blocks * a.kv_heads), a.n_split), kThreads, Shape<HD>::SMEM, ctx->stream>>>(a);
    RLB_LAUNCH_CHECK();
    count_launch(ctx);
    return RLB_OK;
}

}  // namespace

int attn_long_f32_splits(rlb_ctx* ctx, const AttnLongArgs& a) {
    if (ctx->attn_long_splits) return ctx->attn_long_splits;
    // rounds over the SMs times the steps of a split and about two more for its set-up and record
    const int64_t ctas = (int64_t)a.kv_heads * (((int64_t)a.n * a.group + QT - 1) / QT), slots = (int64_t)ctx->sm_count * 2;
    const int64_t seen = std::min<int64_t>((int64_t)a.window + a.sinks + QT / a.group, (int64_t)a.start + a.n), steps = (seen + TK - 1) / TK;
    int64_t best = 1, cost = INT64_MAX;
    for (int64_t s = 1; s <= std::max<int64_t>(1, std::min<int64_t>(steps / 2, std::min<int64_t>(64, record_limit(a)))); s++) {
        const int64_t c = ((ctas * s + slots - 1) / slots) * ((steps + s - 1) / s + 2);
        if (c < cost) { cost = c; best = s; }
    }
    return (int)best;
}

double attn_long_f32_us(rlb_ctx* ctx, const AttnLongArgs& a, int splits) {
    const int64_t ctas = (int64_t)a.kv_heads * (((int64_t)a.n * a.group + QT - 1) / QT), slots = (int64_t)ctx->sm_count * 2;
    const int64_t seen = std::min<int64_t>((int64_t)a.window + a.sinks + QT / a.group, (int64_t)a.start + a.n), steps = (seen + TK - 1) / TK;
    return (splits > 1 ? 10 : 6) + 15.0 * a.hd / 128 * (double)((ctas * splits + slots - 1) / slots) * (double)((steps + splits - 1) / splits);
}

int launch_attn_long_f32(rlb_ctx* ctx, const AttnLongArgs& a) { return a.hd == 128 ? launch<128>(ctx, a) : launch<64>(ctx, a); }
