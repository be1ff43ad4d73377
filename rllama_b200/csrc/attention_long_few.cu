// Long-context attention of few query rows (a generated token, a handful of drafted ones) over f16 and 4-bit caches:
// attention_long.cu says what is computed. The time is that of reading the cache, so every K/V row is fetched once for up to
// eight query rows that share its head (row = i * group + g, as in attention_long_tc.cu).
//
// A CTA takes eight rows of a K/V head and a share of the positions that they see. A warp of its own keeps a ring of stages
// of 128 positions full with bulk copies (neighbouring rows are one piece of memory); each of eight warps takes 16
// positions of a stage:
//  * S (16 x 8 positions, twice) = [q hi; q lo] K^T with mma.sync: the eight queries as two f16 halves each, x = hi + lo, are
//    the 16 rows of the A operand, so the scores carry 22 bits of the queries at no further MMA. A thread's share of K is
//    16 contiguous bytes of a row (or one 4-bit word of every group, cache4.h): the contraction index may be ordered
//    freely as long as the queries are ordered alike.
//  * the weights 2^(s - m + 7) in f16 are then in the right place for the B operand of O^T = V^T P: there V is A, its rows the
//    values, its columns the positions; pairs of positions are interleaved with one byte permutation a register.
// The positions of a tile are dealt to the 2 x 8 columns of S so that a thread's four scores belong to positions c, 4 + c, 8 + c, 12 + c: the
// rows of V that the four threads of a column read side by side are then neighbours in shared memory.
// The running maximum m moves only when a score exceeds it by 2^8, as in attention_long_tc.cu, and a row whose result is a NaN
// although its sum is not is computed again from what it sees alone. Scores, maxima, sums and O are f32; rounded to f16: the weights
// (2^-11) and the result.
//
// Measured: 65536 4-bit positions, 32 heads, one token, 94 us, 3.2 TB/s: 446 instructions for 16 positions of a head (185 of them integer and
// conversions), 61 % of the issue slots; 384 positions 6.4 us a call, 5.1 in a graph. 16384 f16 positions and 4 first tokens, 64 heads on 8,
// 20.5 us, 3.3 TB/s: the second kernel and the ring's first fill are half of it.
//
// Loads straight into registers (two tiles ahead: 141 us, one: 107, of 65536 positions, 32 heads, 4 bits) wait for one another: a warp
// tells its outstanding loads apart by six counters only.
#include <algorithm>

#include "attention_long.h"

using namespace attn_long;

namespace {

constexpr int kRows = 8;    // query rows of a CTA
constexpr int kWarps = 8;
constexpr int kMaxCluster = 8;   // (clusters of 16 find room on few SMs: 35 us where two kernels take 21)
constexpr float kShift = 7.f, kLag = 8.f;

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// d = a b + c with another c than d.
__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1, float c01, float c23) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %11, %11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(c01), "f"(c23));
}
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// The ring: stages of POS positions, [K rows][V rows][K scales][V scales]; 4 bits: two CTAs share an SM.
template <int KIND, int HD, bool CLUSTER> struct Ring {
    static constexpr int POS = kWarps * 16, ROW = KIND == CACHE_Q4 ? HD / 2 : HD * 2, SCALES = KIND == CACHE_Q4 ? HD / 16 : 0;
    static constexpr int THREADS = (kWarps + 1) * 32;
    static constexpr int V = POS * ROW, KD = 2 * POS * ROW, VD = KD + POS * SCALES, STAGE = KD + 2 * POS * SCALES;
    static constexpr int STAGES = (KIND == CACHE_Q4 ? 4 : CLUSTER ? 2 : 3) * 128 / HD;
    static constexpr int MOST = CLUSTER ? kMaxCluster : 1;
    static constexpr size_t RECORD = kRows * HD * 4;                       // [split][row][HD] behind the ring, written by the cluster
    static size_t smem(int splits) { return (size_t)STAGES * STAGE + (CLUSTER ? splits * RECORD : 0); }
};
template <typename T> __device__ __forceinline__ T fetch(const char* p) { return *reinterpret_cast<const T*>(p); }

// A thread's share of K in a tile: two rows, of each HD / 4 values in chunks of eight, 8 (4 i + c) ... `row` points to
// the thread's part of a row.
template <int KIND, int HD> struct KFrag;
template <int HD> struct KFrag<CACHE_F16, HD> {
    uint4 x[2][HD / 32];
    static __device__ __forceinline__ int part(int c) { return 16 * c; }
    __device__ __forceinline__ void load(int nt, const char* row) {
#pragma unroll
        for (int i = 0; i < HD / 32; i++) x[nt][i] = fetch<uint4>(row + 64 * i);
    }
    __device__ __forceinline__ void chunk(int nt, int i, uint32_t (&h)[4]) const { h[0] = x[nt][i].x; h[1] = x[nt][i].y; h[2] = x[nt][i].z; h[3] = x[nt][i].w; }
};
// Of a 4-bit row only the codes: a nibble alone in the low bits of an f16 IS a number, u + 8 times 2^-24 (or 2^-20 for the upper
// nibble of a byte), so one AND makes a pair of operands. The factor 16 goes into the queries, the 8 into the accumulator's
// start, and the scales, one for 32 values, multiply each group's sum afterwards.
template <int HD> struct KFrag<CACHE_Q4, HD> {
    static constexpr int G = HD / kQ4Group;
    uint32_t w[2][G];
    static __device__ __forceinline__ int part(int c) { return c * (HD / 8); }
    __device__ __forceinline__ void load(int nt, const char* row) {
        if constexpr (G == 4) *reinterpret_cast<uint4*>(w[nt]) = fetch<uint4>(row);
        else *reinterpret_cast<uint2*>(w[nt]) = fetch<uint2>(row);
    }
    __device__ __forceinline__ void chunk(int nt, int i, uint32_t (&h)[4]) const {
        const uint32_t x = w[nt][i], y = x >> 8;
        h[0] = x & 0x000F000Fu; h[1] = x & 0x00F000F0u; h[2] = y & 0x000F000Fu; h[3] = y & 0x00F000F0u;
    }
};
// The scales of K at positions c, 4 + c, 8 + c, 12 + c of a tile, where the scores are.
template <int KIND, int HD> struct KScales {
    __device__ __forceinline__ void load(int, const char*) {}
};
template <int HD> struct KScales<CACHE_Q4, HD> {
    __half d[4][HD / kQ4Group];
    __device__ __forceinline__ void load(int i, const char* p) {
        if constexpr (HD == 128) *reinterpret_cast<uint2*>(d[i]) = fetch<uint2>(p);
        else *reinterpret_cast<uint32_t*>(d[i]) = fetch<uint32_t>(p);
    }
};
// A thread's share of V in a tile: positions c, 4 + c, 8 + c, 12 + c, of each HD / 64 chunks of eight values. `dim` is a chunk's
// first value; operands(u): pairs of positions of values 2e (f[e][0], f[e][2]) and 2e + 1 (f[e][1], f[e][3]) of chunk u.
template <int KIND, int HD> struct VFrag;
template <int HD> struct VFrag<CACHE_F16, HD> {
    static constexpr int U = HD / 64;
    uint4 x[4][U];
    static __device__ __forceinline__ int dim(int u, int r) { return 8 * (8 * u + r); }
    static __device__ __forceinline__ int part(int r) { return 16 * r; }
    static __device__ __forceinline__ int scale_part(int) { return 0; }
    __device__ __forceinline__ void load(int i, const char* row, const char*) {
#pragma unroll
        for (int u = 0; u < U; u++) x[i][u] = fetch<uint4>(row + 128 * u);
    }
    __device__ __forceinline__ void operands(int u, uint32_t (&f)[4][4]) const {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t* p0 = reinterpret_cast<const uint32_t*>(&x[0][u]);
            const uint32_t* p1 = reinterpret_cast<const uint32_t*>(&x[1][u]);
            const uint32_t* p2 = reinterpret_cast<const uint32_t*>(&x[2][u]);
            const uint32_t* p3 = reinterpret_cast<const uint32_t*>(&x[3][u]);
            f[e][0] = __byte_perm(p0[e], p1[e], 0x5410);
            f[e][1] = __byte_perm(p0[e], p1[e], 0x7632);
            f[e][2] = __byte_perm(p2[e], p3[e], 0x5410);
            f[e][3] = __byte_perm(p2[e], p3[e], 0x7632);
        }
    }
};
template <int HD> struct VFrag<CACHE_Q4, HD> {
    static constexpr int U = HD / 64, G = HD / kQ4Group;
    uint32_t w[4][U];
    __half d[4][U];
    static __device__ __forceinline__ int dim(int u, int r) { const int x = U * r + u; return 32 * (x % G) + 8 * (x / G); }
    static __device__ __forceinline__ int part(int r) { return 4 * U * r; }
    static __device__ __forceinline__ int scale_part(int r) { return 2 * ((U * r) % G); }   // (a thread's words belong to neighbouring groups)
    __device__ __forceinline__ void load(int i, const char* row, const char* scale) {
        if constexpr (U == 2) {
            *reinterpret_cast<uint2*>(w[i]) = fetch<uint2>(row);
            *reinterpret_cast<uint32_t*>(d[i]) = fetch<uint32_t>(scale);
        } else {
            w[i][0] = fetch<uint32_t>(row);
            d[i][0] = __ushort_as_half(fetch<unsigned short>(scale));
        }
    }
    __device__ __forceinline__ void operands(int u, uint32_t (&f)[4][4]) const {
#pragma unroll
        for (int h = 0; h < 2; h++) {   // positions c, 4 + c, then 8 + c, 12 + c
            const __half2 dd = __halves2half2(d[2 * h][u], d[2 * h + 1][u]);
            __half2 even[4], odd[4];
            q4_pairs(__byte_perm(w[2 * h][u], w[2 * h + 1][u], 0x5410), even);
            q4_pairs(__byte_perm(w[2 * h][u], w[2 * h + 1][u], 0x7632), odd);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                f[e][2 * h] = bits(__hmul2(even[e], dd));
                f[e][2 * h + 1] = bits(__hmul2(odd[e], dd));
            }
        }
    }
};

// Shared memory of another CTA of the cluster.
__device__ __forceinline__ uint32_t cluster_map(const void* p, uint32_t rank) {
    uint32_t x;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(x) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return x;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}
template <int N> __device__ __forceinline__ void async_copy(void* dst, const void* src) {   // 4 or 8 bytes
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void async_arrive(uint64_t* bar) {   // once the thread's copies are there
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// CLUSTER: the splits of a row block form a thread-block cluster and meet in the first one's shared memory.
template <int KIND, int HD, bool CLUSTER>
__global__ void __launch_bounds__(Ring<KIND, HD, CLUSTER>::THREADS, KIND == CACHE_Q4 ? 2 : 1) attn_long_few_kernel(const __grid_constant__ AttnLongArgs a, int* err) {
    typedef Ring<KIND, HD, CLUSTER> Y;
    constexpr int KS = HD / 16, U = VFrag<KIND, HD>::U, STAGES = Y::STAGES;
    extern __shared__ __align__(128) char ring[];
    constexpr int LD = HD + 1;   // (a thread's neighbours in a store are 2 rows or 8 columns away)
    float (*o_s)[kRows][LD] = reinterpret_cast<float (*)[kRows][LD]>(ring);   // [warp], after the loop
    static_assert(kWarps * kRows * LD * 4 <= STAGES * Y::STAGE, "the warps' results fit in the ring");
    float* rec_o = reinterpret_cast<float*>(ring + STAGES * Y::STAGE);
    __shared__ float m_s[kWarps][kRows], l_s[kWarps][kRows];
    __shared__ float2 rec_ml[Y::MOST][kRows];
    __shared__ uint4 q_s[HD / 16][32];   // the queries as A operands, a lane's four registers of a product side by side
    __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES];
    __shared__ int dead_flag;
    __shared__ uint32_t bad;
    volatile int* dead = &dead_flag;
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), r = lane >> 2, c = lane & 3;   // (warp: known to be uniform)
    const int n_rows = a.n * a.group, blocks = (n_rows + kRows - 1) / kRows;
    const int kvh = blockIdx.x / blocks, row0 = (blockIdx.x % blocks) * kRows, rows = min(kRows, n_rows - row0);
    const int pa = a.start + row0 / a.group, pb = a.start + (row0 + rows - 1) / a.group;
    const Run run = visible_run(a, pa, pb);
    int chunk = (run.len + a.n_split - 1) / a.n_split;
    chunk = (chunk + 15) & ~15;
    const int v0 = min(run.len, (int)blockIdx.y * chunk), v1 = min(run.len, v0 + chunk);
    const int64_t base = (int64_t)kvh * a.max_seq;

    // (a CTA's shared memory may be written by its cluster only once that CTA is running)
    if constexpr (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    float o[U][4][4] = {}, m = -FLT_MAX, l = 0.f;
    if (warp == kWarps) {
        // ------------------------------- keeps the ring full ---------------------------------------------------------
        if (lane == 0) {
            dead_flag = 0;
            bad = 0;
            for (int s = 0; s < STAGES; s++) {
                mbar_init(&full[s], KIND == CACHE_Q4 ? 33 : 1);   // the announced bytes, and the scales' 32 threads
                mbar_init(&empty[s], kWarps);
            }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("bar.arrive 1, %0;" ::"n"(Y::THREADS) : "memory");   // the barriers are there; the first copies go out at once
        const char *k = reinterpret_cast<const char*>(a.k) + base * Y::ROW, *v = reinterpret_cast<const char*>(a.v) + base * Y::ROW;
        uint32_t s = 0, phase = 1;
        int p0 = v0, issued = 0;
        for (; p0 < v1; p0 += Y::POS, issued++) {
            if (issued >= STAGES && !warp_wait(&empty[s], phase, dead, err)) break;
            char* dst = ring + s * Y::STAGE;
            const int p1 = min(p0 + Y::POS, v1), cut = min(max(run.s, p0), p1);   // [p0, cut) of the first run, [cut, p1) of the second
            if (lane == 0) {
                mbar_expect_tx(&full[s], (uint32_t)(p1 - p0) * 2 * Y::ROW);
                if (cut > p0) {
                    bulk_load(dst, k + (int64_t)p0 * Y::ROW, (cut - p0) * Y::ROW, &full[s]);
                    bulk_load(dst + Y::V, v + (int64_t)p0 * Y::ROW, (cut - p0) * Y::ROW, &full[s]);
                }
                if (p1 > cut) {
                    const int64_t t = run.at(cut);
                    bulk_load(dst + (cut - p0) * Y::ROW, k + t * Y::ROW, (p1 - cut) * Y::ROW, &full[s]);
                    bulk_load(dst + Y::V + (cut - p0) * Y::ROW, v + t * Y::ROW, (p1 - cut) * Y::ROW, &full[s]);
                }
            }
            if constexpr (KIND == CACHE_Q4) {   // (8 or 4 bytes a row: no 16-byte boundary for a bulk copy to start at)
                for (int x = lane; x < p1 - p0; x += 32) {
                    const int64_t t = base + run.at(p0 + x);
                    async_copy<Y::SCALES>(dst + Y::KD + x * Y::SCALES, reinterpret_cast<const char*>(a.k_scale) + t * Y::SCALES);
                    async_copy<Y::SCALES>(dst + Y::VD + x * Y::SCALES, reinterpret_cast<const char*>(a.v_scale) + t * Y::SCALES);
                }
                async_arrive(&full[s]);
            }
            if (++s == STAGES) { s = 0; phase ^= 1; }
        }
        for (int x = max(0, issued - STAGES); x < issued; x++) mbar_drain(&full[x % STAGES], (x / STAGES) & 1);   // no copy outlives the ring
    } else {
        // the queries: rows r (high halves) and r + 8 (low halves) of the A operand
        const int row = row0 + min(r, rows - 1), p = a.start + row / a.group, low = window_low(a, p);
        float k0[KIND == CACHE_Q4 ? HD / kQ4Group : 1][2] = {};   // -8 times a group's sum of the row's high and low halves, times 2^-24
        float c2;
        bool late = false;   // 4 bits: 2^24 is a factor of its own
        {
            const float* src = a.q + (int64_t)(row / a.group) * a.q_ld + (int64_t)(kvh * a.group + row % a.group) * HD + 8 * c;
            float x[KS][4], top = 0.f;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                *reinterpret_cast<float4*>(x[s]) = *reinterpret_cast<const float4*>(src + 32 * (s >> 1) + 4 * (s & 1));
#pragma unroll
                for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(x[s][e]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // scaled by a power of two so that the row's largest element lies in [2^8, 2^9), whatever its magnitude
            int e = (int)(__float_as_uint(top) >> 23) - 127;
            e = e > 127 ? 0 : max(e, -100);
            const float up = r < rows ? __uint_as_float((uint32_t)(8 - e + 127) << 23) : 0.f;
            c2 = rsqrtf((float)HD) * 1.4426950408889634f * __uint_as_float((uint32_t)(e - 8 + 127) << 23);
#pragma unroll
            for (int s = 0; s < KS; s++) {
                uint32_t q[4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float y0 = x[s][2 * h] * up, y1 = x[s][2 * h + 1] * up;
                    const __half2 hi = __floats2half2_rn(y0, y1);
                    const float2 f = __half22float2(hi);
                    const __half2 lo = __floats2half2_rn(y0 - f.x, y1 - f.y);
                    if constexpr (KIND == CACHE_Q4) {
                        const float2 g = __half22float2(lo);
                        k0[s >> 1][0] += f.x + f.y;
                        k0[s >> 1][1] += g.x + g.y;
                        const __half2 k = __floats2half2_rn(h ? 0.0625f : 1.f, h ? 0.0625f : 1.f);   // (upper nibbles come 16 times as large)
                        q[2 * h] = bits(__hmul2(hi, k));
                        q[2 * h + 1] = bits(__hmul2(lo, k));
                    } else {
                        q[2 * h] = bits(hi);
                        q[2 * h + 1] = bits(lo);
                    }
                }
                if (warp == s % kWarps) q_s[s][lane] = make_uint4(q[0], q[1], q[2], q[3]);
            }
            if constexpr (KIND == CACHE_Q4) {
#pragma unroll
                for (int g = 0; g < HD / kQ4Group; g++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        k0[g][h] += __shfl_xor_sync(0xffffffffu, k0[g][h], 1);
                        k0[g][h] += __shfl_xor_sync(0xffffffffu, k0[g][h], 2);
                        k0[g][h] *= -8.f / 16777216.f;
                    }
                // (with queries from 2^112 on the factor of all would not be finite, although their scores are; then it is applied in two)
                late = __any_sync(0xffffffffu, c2 > 0x1p103f);
                if (!late) c2 *= 16777216.f;
            }
        }
        // the thread's places in a stage
        const int kp = (warp * 16 + (r >> 1) + 4 * (r & 1)) * Y::ROW + KFrag<KIND, HD>::part(c), kd = Y::KD + (warp * 16 + c) * Y::SCALES;
        const int vp = Y::V + (warp * 16 + c) * Y::ROW + VFrag<KIND, HD>::part(r), vd = Y::VD + (warp * 16 + c) * Y::SCALES + VFrag<KIND, HD>::scale_part(r);
        // One tile, at virtual position v; `there`: how many of its positions are in the stage (those behind them read the last one
        // and weigh nothing).
        auto tile = [&](int v, const char* stage, int there) {
            KFrag<KIND, HD> kf;
            KScales<KIND, HD> ks;
            VFrag<KIND, HD> vf;
            if (there >= 16) {
#pragma unroll
                for (int nt = 0; nt < 2; nt++) kf.load(nt, stage + kp + nt * 8 * Y::ROW);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    ks.load(e, stage + kd + e * 4 * Y::SCALES);
                    vf.load(e, stage + vp + e * 4 * Y::ROW, stage + vd + e * 4 * Y::SCALES);
                }
            } else {
#pragma unroll
                for (int nt = 0; nt < 2; nt++) {
                    const int x = (r >> 1) + 4 * (r & 1);
                    kf.load(nt, stage + kp + (min(x + 8 * nt, there - 1) - x) * Y::ROW);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int x = min(4 * e + c, there - 1) - c;
                    ks.load(e, stage + kd + x * Y::SCALES);
                    vf.load(e, stage + vp + x * Y::ROW, stage + vd + x * Y::SCALES);
                }
            }
            float x[4] = {};   // scores of the thread's row at positions c, 4 + c, 8 + c, 12 + c
            if constexpr (KIND == CACHE_Q4) {
#pragma unroll
                for (int g = 0; g < HD / kQ4Group; g++)
#pragma unroll
                    for (int nt = 0; nt < 2; nt++) {
                        uint32_t h[4];
                        float s[4];
                        kf.chunk(nt, g, h);
                        mma16816(s, q_s[2 * g][lane], h[0], h[1], k0[g][0], k0[g][1]);
                        mma16816(s, q_s[2 * g + 1][lane], h[2], h[3]);
#pragma unroll
                        for (int e = 0; e < 2; e++) x[2 * nt + e] = fmaf(__half2float(ks.d[2 * nt + e][g]), s[e] + s[2 + e], x[2 * nt + e]);
                    }
            } else {
                float s[2][4] = {};
#pragma unroll
                for (int i = 0; i < HD / 32; i++)
#pragma unroll
                    for (int nt = 0; nt < 2; nt++) {
                        uint32_t h[4];
                        kf.chunk(nt, i, h);
                        mma16816(s[nt], q_s[2 * i][lane], h[0], h[1]);
                        mma16816(s[nt], q_s[2 * i + 1][lane], h[2], h[3]);
                    }
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = s[e >> 1][e & 1] + s[e >> 1][2 + (e & 1)];
            }
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] *= c2;
            if (KIND == CACHE_Q4 && late) {
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] *= 16777216.f;
            }
            // (a block of one position sees all of its share)
            bool whole = v + 16 <= v1 && (v >= run.s || v + 16 <= run.s);
            if (pa != pb) { const int t0 = run.at(v); whole = whole && t0 + 15 <= pa && (t0 >= window_low(a, pb) || t0 + 15 < a.sinks); }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int w = v + 4 * e + c, t = run.at(w);
                    if (!(w < v1 && t <= p && (t >= low || t < a.sinks))) x[e] = -INFINITY;
                }
            }
            float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            // (no weight reaches 2^16, where f16 ends, whatever the rounding of m + kLag and kShift - m)
            if (__any_sync(0xffffffffu, top >= m + kLag)) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float m_new = fmaxf(m, top), scale = ex2_approx(m - m_new);
                m = m_new;
                l *= scale;
                const float f0 = __shfl_sync(0xffffffffu, scale, 8 * c), f1 = __shfl_sync(0xffffffffu, scale, 8 * c + 4);   // of query rows 2c, 2c + 1
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) { o[u][e][0] *= f0; o[u][e][1] *= f1; o[u][e][2] *= f0; o[u][e][3] *= f1; }
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[e] = ex2_approx(x[e] + (kShift - m));
                l += x[e];
            }
            const uint32_t b0 = bits(__floats2half2_rn(x[0], x[1])), b1 = bits(__floats2half2_rn(x[2], x[3]));
#pragma unroll
            for (int u = 0; u < U; u++) {
                uint32_t f[4][4];
                vf.operands(u, f);
#pragma unroll
                for (int e = 0; e < 4; e++) mma16816(o[u][e], make_uint4(f[e][0], f[e][1], f[e][2], f[e][3]), b0, b1);
            }
        };
        asm volatile("bar.sync 1, %0;" ::"n"(Y::THREADS) : "memory");   // q_s, and the barriers
        uint32_t s = 0, phase = 0;
        for (int p0 = v0; p0 < v1; p0 += Y::POS) {
            if (!warp_wait(&full[s], phase, dead, err)) break;
            const int v = p0 + warp * 16;   // the warp's tile
            if (v < v1) tile(v, ring + s * Y::STAGE, v1 - v);
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
            if (++s == STAGES) { s = 0; phase ^= 1; }
        }
    }
    // the warps' shares, in the ring's room
    __syncthreads();
    if (warp < kWarps) {
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (c == 0) { m_s[warp][r] = m; l_s[warp][r] = l; }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (2 * c + (x & 1) < rows) o_s[warp][2 * c + (x & 1)][VFrag<KIND, HD>::dim(u, r) + 2 * e + (x >> 1)] = o[u][e][x];
    }
    __syncthreads();
    constexpr int PER = kRows * HD / (kWarps * 32);   // values of the result a thread joins: of one row, PER neighbouring columns
    const bool joins = warp < kWarps;
    const int jr = joins ? threadIdx.x * PER / HD : 0, jc = threadIdx.x * PER % HD;
    float M = -FLT_MAX, L = 0.f, O[PER] = {};
    // Joins n partial results of a row.
    auto join = [&](int n, int from) {
        M = -FLT_MAX;
        L = 0.f;
#pragma unroll
        for (int e = 0; e < PER; e++) O[e] = 0.f;
        for (int w = 0; w < n; w++) M = fmaxf(M, m_s[w][from]);
        for (int w = 0; w < n; w++) {
            const float f = ex2_approx(m_s[w][from] - M);
            L = fmaf(l_s[w][from], f, L);
#pragma unroll
            for (int e = 0; e < PER; e++) O[e] = fmaf(o_s[w][from][jc + e], f, O[e]);
        }
    };
    const bool live = joins && jr < rows;
    if (live) join(kWarps, jr);
    M -= kShift;
    float check = 0.f;   // a NaN once one of them is
#pragma unroll
    for (int e = 0; e < PER; e++) check += fabsf(O[e]);
    const int jrow = row0 + min(jr, rows - 1), ji = jrow / a.group, jh = kvh * a.group + jrow % a.group;
    const bool sees = visible_run(a, a.start + ji, a.start + ji).len > 0;
    // A NaN that the sum has too comes from a score that the row sees, and an infinity from a value that it sees: those are the result. Any other may come
    // from a position that it does not see, times weight zero. (A row that sees something has a sum above zero somewhere, but perhaps not in this share.)
    if (live && ((check != check && L == L) || (a.n_split == 1 && sees && L == 0.f))) atomicOr(&bad, 1u << jr);
    __syncthreads();
    for (uint32_t todo = bad; todo; todo &= todo - 1) {   // uniform: rows next to infinite or NaN cache contents that they do not see, one by one
        const int y = __ffs(todo) - 1, again = row0 + y, i = again / a.group, head = kvh * a.group + again % a.group, pp = a.start + i;
        constexpr int N = HD / 32;
        PlainRow<KIND, HD> one(a, i, head, lane);
        for (int w = v0 + warp; joins && w < v1; w += kWarps) {
            const int t = run.at(w);
            if (visible(a, pp, t)) one.see(a, base + t, lane);
        }
        __syncthreads();
        if (joins) {
            if (lane == 0) { m_s[warp][0] = one.m; l_s[warp][0] = one.l; }
#pragma unroll
            for (int e = 0; e < N; e++) o_s[warp][0][lane * N + e] = one.o[e];
        }
        __syncthreads();
        if (jr == y) join(kWarps, 0);
    }
    if constexpr (CLUSTER) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // every CTA of the cluster is running
        if (live) {
            const uint32_t to = cluster_map(rec_o + ((blockIdx.y * kRows + jr) * HD + jc), 0);
            if constexpr (PER == 4)
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(O[0]), "f"(O[1]), "f"(O[PER - 2]), "f"(O[PER - 1]) : "memory");
            else
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(O[0]), "f"(O[1]) : "memory");
            if (jc == 0) {
                const uint32_t ml = cluster_map(&rec_ml[blockIdx.y][jr], 0);
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(ml), "f"(M), "f"(L) : "memory");
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (blockIdx.y != 0 || !live) return;
        M = -FLT_MAX;
        L = 0.f;
#pragma unroll
        for (int e = 0; e < PER; e++) O[e] = 0.f;
        for (int w = 0; w < a.n_split; w++) M = fmaxf(M, rec_ml[w][jr].x);
        for (int w = 0; w < a.n_split; w++) {
            const float2 ml = rec_ml[w][jr];
            const float f = ex2_approx(ml.x - M);
            L = fmaf(ml.y, f, L);
#pragma unroll
            for (int e = 0; e < PER; e++) O[e] = fmaf(rec_o[(w * kRows + jr) * HD + jc + e], f, O[e]);
        }
    }
    if (!live) return;
    if (!CLUSTER && a.n_split > 1) {
        const int64_t rec = ((int64_t)ji * a.heads + jh) * a.n_split + blockIdx.y;
        if constexpr (PER == 4) *reinterpret_cast<float4*>(a.rec_o + rec * HD + jc) = make_float4(O[0], O[1], O[PER - 2], O[PER - 1]);
        else *reinterpret_cast<float2*>(a.rec_o + rec * HD + jc) = make_float2(O[0], O[1]);
        if (jc == 0) a.rec_ml[rec] = make_float2(M, L);
        return;
    }
    const float inv = sees ? 1.0f / L : 0.f;
    __half* dst = reinterpret_cast<__half*>(a.out) + ji * a.out_ld + (int64_t)jh * HD + jc;
#pragma unroll
    for (int e = 0; e < PER; e += 2) {
        const float x = O[e] * inv, y = O[e + 1] * inv;
        // (4-bit values end at 65408: no rounding puts their mean beyond f16)
        *reinterpret_cast<__half2*>(dst + e) = !sees ? __half2half2(__ushort_as_half(0)) : KIND == CACHE_F16 ? mean_f16(x, y) : __floats2half2_rn(x, y);
    }
}

template <int KIND, int HD>
int launch(rlb_ctx* ctx, const AttnLongArgs& a) {
    const int64_t blocks = ((int64_t)a.n * a.group + kRows - 1) / kRows;
    const bool cluster = a.n_split > 1 && a.rec_o == nullptr;
    typedef Ring<KIND, HD, true> YC;
    const size_t smem = cluster ? YC::smem(a.n_split) : Ring<KIND, HD, false>::smem(1), most = cluster ? YC::smem(YC::MOST) : smem;
    auto kern = cluster ? attn_long_few_kernel<KIND, HD, true> : attn_long_few_kernel<KIND, HD, false>;
    static std::atomic<uint64_t> set[2];
    if (!attr_done(set[cluster], ctx->device)) {
        RLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
        attr_mark(set[cluster], ctx->device);
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(blocks * a.kv_heads), a.n_split);
    lc.blockDim = dim3(YC::THREADS);
    lc.dynamicSmemBytes = smem;
    lc.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = (unsigned)a.n_split;
    attr[0].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = cluster ? 1 : 0;
    RLB_CUDA(cudaLaunchKernelEx(&lc, kern, a, ctx->d_err));
    count_launch(ctx);
    return RLB_OK;
}

}  // namespace

// Positions that some row of a block of `rows` rows sees, at most.
static int64_t positions_seen(const AttnLongArgs& a, int rows) {
    return std::min<int64_t>((int64_t)a.window + a.sinks + rows / a.group, (int64_t)a.start + a.n);
}

AttnSplit attn_long_few_splits(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a) {
    if (const int n = ctx->attn_long_splits) return {n, n > 1 && (ctx->attn_long_records || n > kMaxCluster)};
    const int64_t ctas = (int64_t)a.kv_heads * (((int64_t)a.n * a.group + kRows - 1) / kRows), slots = (int64_t)ctx->sm_count * (kind == CACHE_Q4 ? 2 : 1);
    const int64_t seen = positions_seen(a, kRows);
    // as many as fill the SMs, but at least a tile of 16 positions for every warp
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(slots / ctas, 256), (seen + kWarps * 16 - 1) / (kWarps * 16)));
    // A cluster joins its splits through shared memory; more of them need records and a second kernel, which costs about 2 us more, the
    // time of 13 MB. That is weighed against the SMs that a cluster's eight splits leave empty. (One token, 32 heads, 384
    // 4-bit positions: three splits in a cluster 6.8 us, through records 10.6. The last CTA to arrive joining the
    // records, without a second kernel, was no faster than it.)
    const int64_t cluster = std::min<int64_t>(most, kMaxCluster);
    const double bytes = 2.0 * (double)seen * a.kv_heads * (kind == CACHE_Q4 ? a.hd / 2 + a.hd / 16 : a.hd * 2);
    if (bytes * ((double)most / cluster - 1) < 13e6) return {(int)cluster, false};
    return {(int)most, true};
}

// 6 us, 2 more for a second kernel, and the rounds of CTAs over the SMs, a CTA reading 44 KB a us (f16: an SM's share of the memory's rate) or,
// with 4 bits and two CTAs an SM, 9.8 KB (what their arithmetic allows). A round's own cost, whatever it reads, is not counted:
// attention_long.cu says where that matters.
double attn_long_few_us(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a, AttnSplit s) {
    const int64_t ctas = (int64_t)a.kv_heads * (((int64_t)a.n * a.group + kRows - 1) / kRows), slots = (int64_t)ctx->sm_count * (kind == CACHE_Q4 ? 2 : 1);
    const double row = kind == CACHE_Q4 ? a.hd + a.hd / 8 : a.hd * 4, rate = kind == CACHE_Q4 ? 9.8e3 : 44e3;
    return 6 + (s.records ? 2 : 0) + (double)((ctas * s.n + slots - 1) / slots) * (double)positions_seen(a, kRows) / s.n * row / rate;
}

int launch_attn_long_few(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a) {
    if (kind == CACHE_F16) return a.hd == 128 ? launch<CACHE_F16, 128>(ctx, a) : launch<CACHE_F16, 64>(ctx, a);
    return a.hd == 128 ? launch<CACHE_Q4, 128>(ctx, a) : launch<CACHE_Q4, 64>(ctx, a);
}
