// Long-context attention of many query rows on the tensor cores (f16 and 4-bit caches): attention_long.cu says what is
// computed. Query rows that share a K/V head form one list, row = i * group + g, so a tile of 128 rows is full even when a
// few tokens attend with many heads.
//
// A CTA owns 256 rows (two tiles of 128) of a K/V head and walks the positions that some of them see in steps of 128:
//  * K and V steps pass through a ring of shared-memory stages. An f16 cache's are fetched by TMA (128-byte swizzle, the
//    tensor's extent ends at the last visible position: rows behind it read as zeros). A 4-bit cache's are unpacked by
//    four warps; its values are f16 numbers, so the unpacked operand carries no rounding.
//  * one thread issues the MMAs: S = Q K^T (both operands in shared memory), then O += P V with P in tensor memory as the
//    A operand. S, and over it P, and O of both tiles fill the 512 columns. While one tile's scores go through the
//    softmax, the other tile's products run.
//  * eight warps do the softmax, a thread a row: maximum of the step's 128 scores, weights 2^(s - m + 7) rounded to f16
//    (their sum is taken before the rounding), back to tensor memory. The running maximum m is only moved when a row's
//    scores exceed it by 2^8 (then the row's O is scaled in place); weights therefore stay below 2^15, and the factor
//    2^7 keeps weights down to 2^-21 of the largest normal f16 numbers. It cancels in O / l.
//
// Rounded to f16 besides the result: the queries, scaled by a power of two per row so that their largest element lies in
// [2^8, 2^9) whatever the row's magnitude (an error of at most 2^-11 sum |q k| / sqrt(head_dim) in a score), and the
// weights (2^-11 each). Scores, maxima, sums and O are f32.
//
// A zero weight times an infinite or NaN value is a NaN in an MMA, so a row whose result is not finite is computed again,
// one warp to a row, from the positions that it sees alone. Only rows next to such cache contents pay for it.
//
// Every wait is bounded; when one runs out the kernel raises the context's error word, no later wait of the CTA blocks, and
// the tensor memory is released before the CTA returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "attention_long.h"

using namespace attn_long;

namespace {

constexpr int QT = 128;                 // rows of a tile (MMA M)
constexpr int QB = 2 * QT;              // rows of a CTA
constexpr int TK = 128;                 // positions of a step
constexpr int kSoftmaxWarps = 8;
constexpr int kMmaWarp = kSoftmaxWarps;
constexpr int kLoadWarp = kMmaWarp + 1;
constexpr int kUnpackWarps = 4;
constexpr uint32_t kWaitLimit = 1u << 22;
constexpr float kShift = 7.f;           // weights carry 2^7
constexpr float kLag = 8.f;             // the running maximum may lag by 2^8

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
// Waits, with the same limit, for work of the CTA's own that is in flight, whether or not the CTA gave up.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kWaitLimit && !mbar_try_wait(bar, parity); i++) {}
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
// Shared-memory operand descriptors, 128-byte swizzle, groups of 8 rows 1024 bytes apart. K-major: a row is 128 bytes of the
// contraction index. MN-major: a row is 64 output columns of one contraction index; the next 64 columns follow at lead_bytes.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t addr, uint32_t lead_bytes) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)((lead_bytes >> 4) & 0x3FFFu) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {  // A in tensor memory
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&x)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int e = 0; e < 32; e++) x[e] = __uint_as_float(r[e]);
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two f32 in one register pair, one instruction for both.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The steps of a CTA's rows (positions p0 .. p1): the first tokens [0, s) in steps from 0, then [l, p1] in steps from l.
struct Steps {
    int s, l, n_first, n;
    __device__ __forceinline__ int at(int j) const { return j < n_first ? j * TK : l + (j - n_first) * TK; }
};
__device__ __forceinline__ Steps make_steps(const AttnLongArgs& a, int p0, int p1) {
    const Run r = visible_run(a, p0, p1);
    Steps st;
    st.s = r.s; st.l = r.l;
    st.n_first = (r.s + TK - 1) / TK;
    st.n = st.n_first + (p1 + 1 - r.l + TK - 1) / TK;
    return st;
}
// The columns of step j that some row of a tile with positions pa .. pb sees, in whole blocks of 32: [c0, c1). Products and
// softmax leave the others out, so a first step of four tokens costs a quarter and the diagonal its half.
struct Cols {
    int c0, c1;
    __device__ __forceinline__ bool any() const { return c0 < c1; }
};
__device__ __forceinline__ Cols step_cols(const AttnLongArgs& a, const Steps& st, int j, int pa, int pb) {
    const int t0 = st.at(j);
    Cols c;
    if (j < st.n_first) {
        c.c0 = 0;
        c.c1 = min(TK, (st.s - t0 + 31) & ~31);
    } else {
        c.c0 = t0 < a.sinks ? 0 : max(0, window_low(a, pa) - t0) & ~31;
        c.c1 = min(TK, (max(0, pb + 1 - t0) + 31) & ~31);
    }
    return c;
}

// The plain form of one row over steps [j0, j1), by one warp: what the row sees and nothing else.
template <int KIND, int HD>
__device__ __noinline__ void slow_row(const AttnLongArgs& a, int kvh, int row, int j0, int j1, const Steps& st, float& m_out, float& l_out, float (&o)[HD / 32]) {
    constexpr int N = HD / 32;
    const int lane = threadIdx.x & 31, i = row / a.group, head = kvh * a.group + row % a.group, p = a.start + i;
    const float c2 = rsqrtf((float)HD) * 1.4426950408889634f;
    float q[N], m = -FLT_MAX, l = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) { q[e] = a.q[i * a.q_ld + head * HD + lane * N + e] * c2; o[e] = 0.f; }
    for (int j = j0; j < j1; j++)
        for (int x = 0; x < TK; x++) {
            const int t = st.at(j) + x;
            if (!(j < st.n_first ? t < st.s : visible(a, p, t))) continue;
            float k[N], v[N], s = 0.f;
            const int64_t r = (int64_t)kvh * a.max_seq + t;
            load_row<KIND, HD>(a.k, a.k_scale, r, lane, k);
            load_row<KIND, HD>(a.v, a.v_scale, r, lane, v);
#pragma unroll
            for (int e = 0; e < N; e++) s = fmaf(q[e], k[e], s);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            const float m_new = fmaxf(m, s), w = exp2f(s - m_new), scale = exp2f(m - m_new);
            l = l * scale + w;
#pragma unroll
            for (int e = 0; e < N; e++) o[e] = fmaf(o[e], scale, w * v[e]);
            m = m_new;
        }
    m_out = m;
    l_out = l;
}

template <int KIND, int HD> struct Layout {
    static constexpr int NB = HD / 64;                       // 64-column blocks of a row
    static constexpr uint32_t Q_BYTES = QT * HD * 2;
    static constexpr uint32_t STAGE = TK * HD * 2;
    static constexpr int STAGES = HD == 64 ? 8 : 4;         // 128 KB
    static constexpr int THREADS = (kLoadWarp + (KIND == CACHE_Q4 ? kUnpackWarps : 1)) * 32;
    static constexpr size_t SMEM = 2 * Q_BYTES + STAGES * STAGE + 1024;
};

template <int KIND, int HD>
__global__ void __launch_bounds__(Layout<KIND, HD>::THREADS, 1)
    attn_long_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ CUtensorMap tm_k_first, const __grid_constant__ CUtensorMap tm_v_first, const __grid_constant__ AttnLongArgs a, int* err) {
    typedef Layout<KIND, HD> Y;
    constexpr int NB = Y::NB, STAGES = Y::STAGES;
    constexpr uint32_t TMEM_COLS = 512, O_COL = 2 * TK;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* q_s = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);  // [tile][HD/64][128][64]
    unsigned char* ring = q_s + 2 * Y::Q_BYTES;                                                              // [stage][HD/64][128][64]
    __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], s_full[2], p_ready[2], pv_done[2], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int dead_flag;
    volatile int* dead = &dead_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.x % a.kv_heads;
    const int n_rows = a.n * a.group;
    const int row0 = ((n_rows + QB - 1) / QB - 1 - (int)blockIdx.x / a.kv_heads) * QB;  // the longest rows first
    const int row_last = min(n_rows, row0 + QB) - 1;
    const Steps st = make_steps(a, a.start + row0 / a.group, a.start + row_last / a.group);
    const int per = (st.n + a.n_split - 1) / a.n_split;
    const int j0 = min(st.n, (int)blockIdx.y * per), j1 = min(st.n, j0 + per);
    int pa[2], pb[2];  // first and last position of each tile's rows
#pragma unroll
    for (int t = 0; t < 2; t++) {
        pa[t] = a.start + min(row0 + t * QT, row_last) / a.group;
        pb[t] = a.start + min(row0 + t * QT + QT - 1, row_last) / a.group;
    }
    const bool two = row0 + QT <= row_last;  // the second tile has rows
    auto cols = [&](int t, int j) { return t == 0 || two ? step_cols(a, st, j, pa[t], pb[t]) : Cols{0, 0}; };

    if (threadIdx.x == 0) {
        dead_flag = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&full[s], KIND == CACHE_Q4 ? kUnpackWarps : 1);
            mbar_init(&empty[s], 1);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_ready[t], 4);
            mbar_init(&pv_done[t], 1);
        }
        mbar_init(&drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // The queries as f16 in the A operand's layout: row r, 16-byte chunk c of a 64-column block at r * 128 + ((c ^ (r & 7)) * 16).
    const int tile = warp >> 2, r = threadIdx.x & (QT - 1);   // (softmax threads: their tile and row)
    const int row = min(row0 + tile * QT + r, row_last);
    float c2 = 0.f;                                           // scores are s * c2 in units of log2 e
    if (warp < kSoftmaxWarps) {
        const bool live = row0 + tile * QT + r <= row_last;
        const float4* src = reinterpret_cast<const float4*>(a.q + (int64_t)(row / a.group) * a.q_ld + (int64_t)(kvh * a.group + row % a.group) * HD);
        float top = 0.f;
        for (int c = 0; c < HD / 4; c++) {
            const float4 v = src[c];
            top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
        // 2^e <= top < 2^(e+1); an infinite top keeps its factor (the row is not finite and is computed again)
        int e = (int)((__float_as_uint(top) >> 23) & 0xff) - 127;
        e = e > 127 ? 0 : max(e, -100);
        const float up = live ? __uint_as_float((uint32_t)(8 - e + 127) << 23) : 0.f, down = __uint_as_float((uint32_t)(e - 8 + 127) << 23);
        c2 = rsqrtf((float)HD) * 1.4426950408889634f * down;
        for (int c = 0; c < HD / 8; c++) {
            const float4 v0 = src[2 * c], v1 = src[2 * c + 1];
            __half2 h[4] = {__floats2half2_rn(v0.x * up, v0.y * up), __floats2half2_rn(v0.z * up, v0.w * up), __floats2half2_rn(v1.x * up, v1.y * up),
                            __floats2half2_rn(v1.z * up, v1.w * up)};
            *reinterpret_cast<uint4*>(q_s + tile * Y::Q_BYTES + (c >> 3) * (QT * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = *reinterpret_cast<uint4*>(h);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the MMA reads these through the async proxy
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = tmem_slot;

    if (warp >= kLoadWarp) {
        // ------------------------------- K and V steps into the ring: K(j0), V(j0), K(j0 + 1), ... -------------------
        const int items = 2 * (j1 - j0);
        if constexpr (KIND == CACHE_F16) {
            if (lane == 0) {
                int x = 0;
                for (; x < items; x++) {
                    const int s = x % STAGES, j = j0 + x / 2, t0 = st.at(j);
                    const CUtensorMap* map = j < st.n_first ? ((x & 1) ? &tm_v_first : &tm_k_first) : ((x & 1) ? &tm_v : &tm_k);
                    if (x >= STAGES && !mbar_wait(&empty[s], (x / STAGES - 1) & 1, dead, err)) break;
                    mbar_expect_tx(&full[s], Y::STAGE);
#pragma unroll
                    for (int b = 0; b < NB; b++) tma_load_3d(ring + s * Y::STAGE + b * (TK * 128), map, b * 64, t0, kvh, &full[s]);
                }
                for (int y = max(0, x - STAGES); y < x; y++) mbar_drain(&full[y % STAGES], (y / STAGES) & 1);  // no copy outlives the CTA
            }
        } else {
            // A thread unpacks a quarter of a row: the same block of eight values of every group (cache4.h). 32 rows a pass.
            constexpr int G = HD / kQ4Group;
            const int x0 = threadIdx.x - kLoadWarp * 32, quarter = x0 & 3, rr = x0 >> 2;
            uint32_t w[4][G];
            __half d[4][G];
            auto fetch = [&](int x) {
                const int j = j0 + x / 2, t0 = st.at(j), end = j < st.n_first ? min(a.sinks, a.start + a.n) : a.start + a.n;
                const uint8_t* codes = reinterpret_cast<const uint8_t*>((x & 1) ? a.v : a.k);
                const __half* scales = (x & 1) ? a.v_scale : a.k_scale;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int t = t0 + u * 32 + rr;
                    const int64_t at = (int64_t)kvh * a.max_seq + t;
                    if (t < end) {
                        if constexpr (G == 4) {
                            *reinterpret_cast<uint4*>(w[u]) = *reinterpret_cast<const uint4*>(codes + at * 64 + quarter * 16);
                            *reinterpret_cast<uint2*>(d[u]) = *reinterpret_cast<const uint2*>(scales + at * 4);
                        } else {
                            *reinterpret_cast<uint2*>(w[u]) = *reinterpret_cast<const uint2*>(codes + at * 32 + quarter * 8);
                            *reinterpret_cast<uint32_t*>(d[u]) = *reinterpret_cast<const uint32_t*>(scales + at * 2);
                        }
                    } else {
#pragma unroll
                        for (int g = 0; g < G; g++) { w[u][g] = 0; d[u][g] = __ushort_as_half(0); }
                    }
                }
            };
            if (items > 0) fetch(0);
            for (int x = 0; x < items; x++) {
                const int s = x % STAGES;
                if (x >= STAGES && !mbar_wait(&empty[s], (x / STAGES - 1) & 1, dead, err)) break;
                unsigned char* dst = ring + s * Y::STAGE;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int y = u * 32 + rr;
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        const __half2 dd = __half2half2(d[u][g]);
                        __half2 h[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) h[e] = __hmul2(q4_pair(w[u][g], e), dd);
                        const int chunk = 4 * g + quarter;   // eight values 32 g + 8 quarter ...
                        *reinterpret_cast<uint4*>(dst + (chunk >> 3) * (TK * 128) + y * 128 + (((chunk & 7) ^ (y & 7)) << 4)) = *reinterpret_cast<uint4*>(h);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
                if (x + 1 < items) fetch(x + 1);
            }
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------- MMA issuer ------------------------------------------------------------------
        if (lane == 0) {
            const uint32_t idesc_s = (1u << 4) | ((uint32_t)(QT >> 4) << 24);   // | N / 8 << 17
            const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(QT >> 4) << 24);
            uint32_t done[2] = {0, 0};   // output products issued
            auto scores = [&](int t, int j, Cols c) {
                const uint32_t qa = smem_u32(q_s) + t * Y::Q_BYTES, kb = smem_u32(ring) + (uint32_t)((2 * (j - j0)) % STAGES) * Y::STAGE + c.c0 * 128;
                const uint32_t id = idesc_s | (uint32_t)((c.c1 - c.c0) >> 3) << 17;
#pragma unroll
                for (int k = 0; k < HD / 16; k++)
                    umma_ss(tmem + t * TK + c.c0, desc_kmajor(qa + (k >> 2) * (QT * 128) + (k & 3) * 32), desc_kmajor(kb + (k >> 2) * (TK * 128) + (k & 3) * 32), id, k > 0);
                umma_commit(&s_full[t]);
            };
            auto wait_item = [&](int x) { return mbar_wait(&full[x % STAGES], (x / STAGES) & 1, dead, err); };
            bool ok = j1 > j0 && wait_item(0);
            if (ok) {
                tc_after();
                for (int t = 0; t < 2; t++)
                    if (const Cols c = cols(t, j0); c.any()) scores(t, j0, c);
                umma_commit(&empty[0]);
            }
            for (int j = j0; j < j1 && ok; j++) {
                const int xv = 2 * (j - j0) + 1;
                for (int t = 0; t < 2 && ok; t++) {
                    const Cols now = cols(t, j);
                    if (t == 0) ok = wait_item(xv);
                    if (now.any() && ok) {
                        ok = mbar_wait(&p_ready[t], done[t] & 1, dead, err);
                        if (!ok) break;
                        tc_after();
                        const uint32_t vb = smem_u32(ring) + (uint32_t)(xv % STAGES) * Y::STAGE;
                        for (int k = now.c0 / 16; k < now.c1 / 16; k++)
                            umma_ts(tmem + O_COL + t * HD, tmem + t * TK + k * 8, desc_mnmajor(vb + k * 2048, TK * 128), idesc_o, done[t] > 0 || k > now.c0 / 16);
                        umma_commit(&pv_done[t]);
                        done[t]++;
                    }
                    if (t == 1) umma_commit(&empty[xv % STAGES]);
                    if (j + 1 < j1) {
                        if (t == 0) ok = ok && wait_item(xv + 1);
                        // the scores overwrite the weights: the output product that reads them must be complete
                        if (const Cols next = cols(t, j + 1); ok && next.any()) {
                            ok = done[t] == 0 || mbar_wait(&pv_done[t], (done[t] - 1) & 1, dead, err);
                            if (!ok) break;
                            tc_after();
                            scores(t, j + 1, next);
                        }
                        if (t == 1) umma_commit(&empty[(xv + 1) % STAGES]);
                    }
                }
            }
            if (!ok) {  // no product outlives the CTA either (after a full run the softmax warps have waited for the last)
                umma_commit(&drained);
                mbar_drain(&drained, 0);
            }
        }
    } else {
        // ------------------------------- softmax: a thread owns a row ------------------------------------------------
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + lanes + tile * TK, o_addr = tmem + lanes + O_COL + tile * HD;
        const int p = a.start + row / a.group, low = window_low(a, p);
        float m = -FLT_MAX, l = 0.f;
        uint32_t steps = 0;
        bool ok = true;
        const int warp_row = row0 + tile * QT + (warp & 3) * 32;   // the warp's first and last position
        const int wa = a.start + min(warp_row, row_last) / a.group, wb = a.start + min(warp_row + 31, row_last) / a.group;
        const int low_wa = window_low(a, wa), low_wb = window_low(a, wb);
        for (int j = j0; j < j1 && ok; j++) {
            const Cols now = cols(tile, j);
            if (!now.any()) continue;
            ok = mbar_wait(&s_full[tile], steps & 1, dead, err);
            if (!ok) break;
            tc_after();
            // columns of the step that the row sees: below `to`, and from `from` on or below `first`
            const int t0 = st.at(j);
            const bool in_first = j < st.n_first;
            const int to = (in_first ? st.s : p + 1) - t0, from = (in_first ? 0 : low) - t0, first = (in_first ? 0 : a.sinks) - t0;
            // 0: nobody in the warp sees any of the block of 32 columns, 2: everybody sees all of it, 1: else
            auto block = [&](int c) {
                if (c < now.c0 || c >= now.c1) return -1;
                if (in_first) return c + 32 <= to ? 2 : 1;
                if (c >= wb + 1 - t0 || (c + 32 <= low_wa - t0 && c >= first)) return 0;
                return c + 32 <= wa + 1 - t0 && (c >= low_wb - t0 || c + 32 <= first) ? 2 : 1;
            };
            auto mask = [&](int c, float (&x)[32]) {
#pragma unroll
                for (int e = 0; e < 32; e++) x[e] = (c + e < to && (c + e >= from || c + e < first)) ? x[e] : -INFINITY;
            };
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < TK; c += 32) {
                const int b = block(c);
                if (b <= 0) continue;
                float x[32];
                tmem_ld32(s_addr + c, x);
                if (b == 1) mask(c, x);
#pragma unroll
                for (int e = 0; e < 32; e++) top = fmaxf(top, x[e]);
            }
            top *= c2;
            const bool move = top > m + kLag;
            if (__any_sync(0xffffffffu, move)) {
                const float m_new = move ? top : m, scale = ex2_approx(m - m_new);
                m = m_new;
                l *= scale;
                if (steps > 0) {   // (the previous output product is complete: its completion went before these scores)
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        float x[32];
                        tmem_ld32(o_addr + c, x);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t y[16];
#pragma unroll
                            for (int e = 0; e < 16; e++) y[e] = __float_as_uint(x[h * 16 + e] * scale);
                            tmem_st16(o_addr + c + h * 16, y);
                        }
                    }
                    tmem_st_wait();
                }
            }
            const float shift = kShift - m;
            const uint64_t c2_2 = pack2(c2, c2), shift_2 = pack2(shift, shift);
            uint64_t sum = 0;   // (0, 0)
#pragma unroll
            for (int c = 0; c < TK; c += 32) {
                const int b = block(c);
                if (b < 0) continue;
                uint32_t y[16];
                if (b == 0) {
#pragma unroll
                    for (int e = 0; e < 16; e++) y[e] = 0;
                } else {
                    float x[32];
                    tmem_ld32(s_addr + c, x);
                    if (b == 1) mask(c, x);
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        float w0, w1;
                        unpack2(fma2(pack2(x[2 * e], x[2 * e + 1]), c2_2, shift_2), w0, w1);
                        w0 = ex2_approx(w0);
                        w1 = ex2_approx(w1);
                        sum = add2(sum, pack2(w0, w1));
                        const __half2 h = __floats2half2_rn(w0, w1);
                        y[e] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                }
                tmem_st16(s_addr + c / 2, y);   // over scores that have been read
            }
            float sum0, sum1;
            unpack2(sum, sum0, sum1);
            l += sum0 + sum1;
            tmem_st_wait();
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[tile]);
            steps++;
        }
        if (ok && steps > 0) ok = mbar_wait(&pv_done[tile], (steps - 1) & 1, dead, err);
        const bool live = row0 + tile * QT + r <= row_last;
        if (ok && __any_sync(0xffffffffu, live)) {
            tc_after();
            const int64_t rec = ((int64_t)row / a.group * a.heads + kvh * a.group + row % a.group) * a.n_split + blockIdx.y;
            __half* dst = reinterpret_cast<__half*>(a.out) + (int64_t)(row / a.group) * a.out_ld + (int64_t)(kvh * a.group + row % a.group) * HD;
            const bool empty_row = p + 1 - low + min(a.sinks, low) == 0;
            const float inv = empty_row ? 0.f : 1.0f / l;
            float check = fmaf(l, 0.f, a.n_split == 1 ? inv * 0.f : 0.f);   // a NaN once anything is not finite
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                float x[32];
                if (steps > 0) {
                    tmem_ld32(o_addr + c, x);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) x[e] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < 32; e++) check = fmaf(x[e], 0.f, check);
                if (live && a.n_split > 1) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(a.rec_o + rec * HD + c + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                } else if (live) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        __half2 h[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) h[u] = empty_row ? __half2half2(__ushort_as_half(0)) : __floats2half2_rn(x[e + 2 * u] * inv, x[e + 2 * u + 1] * inv);
                        *reinterpret_cast<uint4*>(dst + c + e) = *reinterpret_cast<uint4*>(h);
                    }
                }
                __syncwarp();
            }
            if (live && a.n_split > 1) a.rec_ml[rec] = make_float2(m - kShift, l);
            // rows next to infinite or NaN cache contents, again and one by one
            uint32_t bad = __ballot_sync(0xffffffffu, live && check != 0.f && !empty_row);
            while (bad) {
                const int b = __ffs(bad) - 1;
                bad &= bad - 1;
                const int again = __shfl_sync(0xffffffffu, row, b);
                float o[HD / 32], sm, sl;
                slow_row<KIND, HD>(a, kvh, again, j0, j1, st, sm, sl, o);
                const int i = again / a.group, head = kvh * a.group + again % a.group;
                const int64_t rb = ((int64_t)i * a.heads + head) * a.n_split + blockIdx.y;
#pragma unroll
                for (int e = 0; e < HD / 32; e++) {
                    const int c = lane * (HD / 32) + e;
                    if (a.n_split > 1) a.rec_o[rb * HD + c] = o[e];
                    else reinterpret_cast<__half*>(a.out)[i * a.out_ld + head * HD + c] = __float2half_rn(o[e] / sl);
                }
                if (a.n_split > 1 && lane == 0) a.rec_ml[rb] = make_float2(sm, sl);
            }
        }
    }
    tc_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 f = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult res;
        cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &res);
        return e == cudaSuccess && res == cudaDriverEntryPointSuccess ? (PFN_cuTensorMapEncodeTiled_v12000)fn : nullptr;
    }();
    return f;
}

// The cache as [kv_heads][positions][hd], positions up to the last that any row of the call sees (or the last of the first
// tokens), so that no row behind it reaches a product; a box is 64 columns of TK positions.
int cache_map(CUtensorMap* map, const void* cache, const AttnLongArgs& a, int positions) {
    if (!encoder()) return rlb_fail(RLB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[3] = {(cuuint64_t)a.hd, (cuuint64_t)positions, (cuuint64_t)a.kv_heads};
    cuuint64_t strides[2] = {(cuuint64_t)a.hd * 2, (cuuint64_t)a.max_seq * a.hd * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)TK, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = encoder()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(cache), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return rlb_fail(RLB_ERR_CUDA, "cuTensorMapEncodeTiled (KV cache) failed with code %d", (int)r);
    return RLB_OK;
}

template <int KIND, int HD>
int launch(rlb_ctx* ctx, const AttnLongArgs& a) {
    typedef Layout<KIND, HD> Y;
    CUtensorMap mk{}, mv{}, mkf{}, mvf{};
    if (KIND == CACHE_F16) {
        const int end = a.start + a.n, first = std::min(a.sinks, end);
        RLB_TRY(cache_map(&mk, a.k, a, end));
        RLB_TRY(cache_map(&mv, a.v, a, end));
        if (first > 0) {
            RLB_TRY(cache_map(&mkf, a.k, a, first));
            RLB_TRY(cache_map(&mvf, a.v, a, first));
        }
    }
    auto kern = attn_long_tc_kernel<KIND, HD>;
    static std::atomic<uint64_t> set{0};
    if (!attr_done(set, ctx->device)) {
        RLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Y::SMEM));
        attr_mark(set, ctx->device);
    }
    const int blocks = (a.n * a.group + QB - 1) / QB;
    kern<<<dim3((unsigned)(blocks * a.kv_heads), a.n_split), Y::THREADS, Y::SMEM, ctx->stream>>>(mk, mv, mkf, mvf, a, ctx->d_err);
    RLB_LAUNCH_CHECK();
    count_launch(ctx);
    return RLB_OK;
}

}  // namespace

int attn_long_tc_splits(rlb_ctx* ctx, const AttnLongArgs& a) {
    // one CTA an SM; a split has at least four steps (its own set-up and record cost about two)
    const int64_t ctas = (int64_t)a.kv_heads * ((a.n * a.group + QB - 1) / QB);
    const int64_t seen = std::min<int64_t>((int64_t)a.window + a.sinks + QB / a.group, (int64_t)a.start + a.n);
    const int64_t steps = (seen + TK - 1) / TK;
    return (int)std::max<int64_t>(1, std::min<int64_t>(ctx->sm_count / std::max<int64_t>(ctas, 1), steps / 4));
}

int launch_attn_long_tc(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a) {
    if (kind == CACHE_F16) return a.hd == 128 ? launch<CACHE_F16, 128>(ctx, a) : launch<CACHE_F16, 64>(ctx, a);
    return a.hd == 128 ? launch<CACHE_Q4, 128>(ctx, a) : launch<CACHE_Q4, 64>(ctx, a);
}
