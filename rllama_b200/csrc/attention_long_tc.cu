// Long-context attention of many query rows on the tensor cores (f16 and 4-bit caches): attention_long.cu says what is
// computed. Query rows that share a K/V head form one list, row = i * group + g, so a tile of 128 rows is full even when a
// few tokens attend with many heads.
//
// A CTA owns one tile of 128 rows of a K/V head (f16; two CTAs share an SM) or two (4 bits) and walks the positions that some of them see in
// steps of 64:
//  * K and V steps pass through a ring of shared-memory stages (attention_long_ring.h), in the order in which they are used: K0 K1 V0 K2 V1 K3 ...
//    An f16 cache's are fetched by TMA (128-byte swizzle, the tensor's extent ends at the last visible position: rows
//    behind it read as zeros). A 4-bit cache's are unpacked by eight warps; its values are f16 numbers, so the unpacked
//    operand carries no rounding.
//  * two warps a tile issue its MMAs: one S = Q K^T (both operands in shared memory; the queries as two f16 halves, x = high + low, one
//    after the other), one O += P V with P in tensor memory as the A operand. Tensor memory holds, per tile, O, one buffer of 64 scores and two of 64 weights: the scores are free
//    again as soon as the softmax has them in registers, so the next ones are computed during the exponentials, and a
//    weight buffer is only needed again two steps later. Neither side waits for a chain of the other's. (Weights written
//    over their scores made a step's chain softmax, output product, next scores: with one buffer of 128 scores 5200
//    cycles for 256 x 128 scores, with two of 64 still 4000.)
//  * four warps a tile do the softmax, a thread a row: maximum of the step's 64 scores, weights 2^(s - m + 7) rounded to f16
//    (their sum is taken before the rounding), back to tensor memory. The running maximum m is only moved when a row's
//    scores exceed it by 2^8 (then the row's O is scaled in place); weights therefore stay below 2^15, and the factor
//    2^7 keeps weights down to 2^-21 of the largest normal f16 numbers. It cancels in O / l.
//
// Measured over repeated calls: 8192 rows, 32 heads on 8, window 2048 and 16 first tokens, 372 us, 652 TFLOP/s, at the clock that the power limit
// leaves (320 us in a graph); 1792 rows, 64 heads, window 512 and 4 first tokens, 80 us, 325 TFLOP/s (70.6 in a graph); 512 rows after 7680
// positions in 4 bits, 40 heads, 150 us, 553 TFLOP/s (140 in a graph; products of the low halves not counted). Two things bound it by turns: the products, of which the
// scores' read both operands from shared memory (6 KB for 32 cycles of arithmetic; leaving their second half out takes the 8192-row prompt from 320 to 256 us),
// and latency, since a step of the softmax is 64 exponentials (512 of its cycles, twice that for the two tiles of an SM) between waits, tensor-memory reads and
// writes of 100 to 200 cycles each. What did not shorten it: part of the exponentials by a polynomial, two threads a row, fetching the next scores before the
// weights are known to have arrived; two f16 tiles a CTA over one ring of six stages (window prompt 79 us where it is 70 in a graph).
//
// Rounded to f16 besides the result: the weights (2^-11 each). Scores, maxima, sums and O are f32. The queries are scaled by a power of two per row so
// that their largest element lies in [2^8, 2^9) whatever the row's magnitude, and their two halves hold 22 bits of it. With the high halves alone a score was
// off by up to 2^-11 sum |q k| / sqrt(head_dim), and results by twice what their own rounding is (4.4e-4 from 64 bits, now 2.9e-4); the low ones double the score
// products and take a stage of the ring (8192-row prompt 253 us in a graph, now 320; 1792-row window prompt 62.6 and 70.6; 512-row 4-bit chunk 132.5 and 139.7).
//
// A zero weight times an infinite or NaN value is a NaN in an MMA, so a row whose result is a NaN although its sum is not is computed
// again, one warp to a row, from the positions that it sees alone. Only rows next to such cache contents pay for it.
//
// Every wait is bounded; when one runs out the kernel raises the context's error word, no later wait of the CTA blocks, and
// the tensor memory is released before the CTA returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "attention_long.h"
#include "attention_long_ring.h"

using namespace attn_long;

namespace {

constexpr int QT = 128;                 // rows of a tile (MMA M)
constexpr int TK = 64;                  // positions of a step
constexpr float kShift = 7.f;           // weights carry 2^7
constexpr float kLag = 8.f;             // the running maximum may lag by 2^8

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
// A thread's own 16-byte aligned piece of shared memory to global memory; the piece is free again on return.
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
    asm volatile("fence.proxy.async.shared::cta;\n cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n cp.async.bulk.commit_group;\n cp.async.bulk.wait_group.read 0;" ::"l"(dst),
                 "r"(smem_u32(src)), "r"(bytes)
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
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 32 columns of the thread's lane. The values are there only after tmem_ld_wait, and `tmem_arrived` on them after it keeps
// the compiler from using them before.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t addr, float* x) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]), "=f"(x[9]), "=f"(x[10]),
          "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15]), "=f"(x[16]), "=f"(x[17]), "=f"(x[18]), "=f"(x[19]), "=f"(x[20]),
          "=f"(x[21]), "=f"(x[22]), "=f"(x[23]), "=f"(x[24]), "=f"(x[25]), "=f"(x[26]), "=f"(x[27]), "=f"(x[28]), "=f"(x[29]), "=f"(x[30]), "=f"(x[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_arrived(float* x) {
#pragma unroll
    for (int e = 0; e < 32; e++) asm volatile("" : "+f"(x[e]));
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&x)[32]) {
    tmem_ld32_issue(addr, x);
    tmem_ld_wait();
    tmem_arrived(x);
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&x)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]), "=f"(x[9]), "=f"(x[10]),
          "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15])
        : "r"(addr));
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; e++) asm volatile("" : "+f"(x[e]));
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

// One row over steps [j0, j1), by one warp: what the row sees and nothing else.
template <int KIND, int HD>
__device__ __noinline__ void slow_row(const AttnLongArgs& a, int kvh, int row, int j0, int j1, const Steps& st, float& m_out, float& l_out, float (&o)[HD / 32]) {
    const int lane = threadIdx.x & 31, i = row / a.group, p = a.start + i;
    PlainRow<KIND, HD> one(a, i, kvh * a.group + row % a.group, lane);
    for (int j = j0; j < j1; j++)
        for (int x = 0; x < TK; x++) {
            const int t = st.at(j) + x;
            if (j < st.n_first ? t < st.s : visible(a, p, t)) one.see(a, (int64_t)kvh * a.max_seq + t, lane);
        }
    m_out = one.m;
    l_out = one.l;
#pragma unroll
    for (int e = 0; e < HD / 32; e++) o[e] = one.o[e];
}

// With head_dim 128, as many stages as fit beside the queries.
template <int KIND, int HD> struct RingOf;
template <> struct RingOf<CACHE_F16, 128> { typedef KvRing<2, 1> T; };
template <> struct RingOf<CACHE_F16, 64> { typedef KvRing<4, 4> T; };
template <> struct RingOf<CACHE_Q4, 128> { typedef KvRing<3, 3> T; };
template <> struct RingOf<CACHE_Q4, 64> { typedef KvRing<8, 8> T; };

template <int KIND, int HD> struct Layout {
    // An f16 CTA has one tile, and two CTAs share an SM: one's first loads, masks and last stores fall into the other's main
    // loop (8192 rows of 32 heads, window 2048: two tiles in one CTA 326 us, two CTAs 278). Unpacking 4-bit rows costs too much to be done for one tile: two share it.
    static constexpr int TILES = KIND == CACHE_Q4 ? 2 : 1;
    static constexpr int ROWS = TILES * QT;                  // rows of a CTA
    static constexpr int NB = HD / 64;                       // 64-column blocks of a row
    // A tile's queries, 128 rows of f16 one after the other, their high halves and then the low ones, and in the end its results, in rows that are 16
    // bytes longer (32 lanes that store 16 bytes of a row each then meet no bank twice).
    static constexpr uint32_t Q_HALF = QT * HD * 2, Q_ROOM = 2 * Q_HALF, OUT_ROW = HD * 2 + 16;
    static_assert(QT * OUT_ROW <= Q_ROOM, "the results fit in the queries' room");
    static constexpr uint32_t STAGE = TK * HD * 2;
    typedef typename RingOf<KIND, HD>::T Ring;
    static constexpr int STAGES = Ring::STAGES;
    static constexpr uint32_t TMEM_COLS = TILES * 256;
    // warps: four a tile for the softmax, two a tile for its MMAs, then one that loads (and an idle one: registers are dealt to four warps
    // at a time), or eight that unpack
    static constexpr int SOFTMAX_WARPS = 4 * TILES, MMA_WARP = SOFTMAX_WARPS, LOAD_WARP = MMA_WARP + 2 * TILES;
    static constexpr int THREADS = (LOAD_WARP + (KIND == CACHE_Q4 ? 8 : 2)) * 32;
    struct Control {   // behind the queries and the ring
        uint64_t full[STAGES], empty[STAGES], s_full[2], s_read[2], drained[4];
        uint64_t p_ready[4], pv_done[4];   // [tile][buffer]: a phase is seen before the next one begins
        float c2[ROWS];                    // a row's scores are s * c2 in units of log2 e
        uint32_t tmem_slot;
        int dead;
    };
    static constexpr size_t SMEM = TILES * Q_ROOM + STAGES * STAGE + sizeof(Control);
    static_assert((2 / TILES) * (SMEM + 1024) <= 228 * 1024, "the CTAs of an SM fit in its shared memory");
    // A thread is launched with LAUNCH_REGS registers (65536 over the threads of an SM, in eights); the MMA and loading warps give theirs to the
    // softmax warps, whose sum with what is left is what was launched: 128 * 152 + 128 * 104 = 256 * 128 (f16), 256 * 120 + 384 * 80 = 640 * 96.
    static constexpr int LAUNCH_REGS = KIND == CACHE_Q4 ? 96 : 128, SOFTMAX_REGS = KIND == CACHE_Q4 ? 120 : 152, OTHER_REGS = KIND == CACHE_Q4 ? 80 : 104;
    static_assert(SOFTMAX_WARPS * SOFTMAX_REGS + (THREADS / 32 - SOFTMAX_WARPS) * OTHER_REGS <= THREADS / 32 * LAUNCH_REGS, "the shares fit in the launch's registers");
    static_assert(MMA_WARP % 4 == 0 && THREADS % 128 == 0, "whole warpgroups give registers away, and whole ones take them");
    static_assert((2 / TILES) * THREADS * LAUNCH_REGS <= 65536, "the CTAs of an SM fit in its registers");
};

template <int KIND, int HD>
__global__ void __launch_bounds__(Layout<KIND, HD>::THREADS, 2 / Layout<KIND, HD>::TILES)
    attn_long_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ CUtensorMap tm_k_first, const __grid_constant__ CUtensorMap tm_v_first, const __grid_constant__ AttnLongArgs a, int ahead, int* err) {
    typedef Layout<KIND, HD> Y;
    typedef typename Y::Ring Ring;
    constexpr int NB = Y::NB, STAGES = Y::STAGES, TILES = Y::TILES, QB = Y::ROWS;
    constexpr uint32_t O_COL = TILES * 2 * TK;   // [tile]: S [TK], P [buffer][TK / 2]; then [tile]: O [HD]
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* q_s = smem;                         // [tile][half][HD/64][128][64]
    unsigned char* ring = q_s + TILES * Y::Q_ROOM;   // [stage][HD/64][64][64]
    typename Y::Control& ctl = *reinterpret_cast<typename Y::Control*>(ring + STAGES * Y::STAGE);
    uint64_t (&full)[STAGES] = ctl.full, (&empty)[STAGES] = ctl.empty, (&s_full)[2] = ctl.s_full, (&s_read)[2] = ctl.s_read, (&drained)[4] = ctl.drained;
    uint64_t (&p_ready)[4] = ctl.p_ready, (&pv_done)[4] = ctl.pv_done;
    float (&c2_s)[QB] = ctl.c2;
    volatile int* dead = &ctl.dead;
    if (smem_u32(smem) & 1023) {   // (the operands' swizzle counts from there; without static shared memory it is where the block's memory begins)
        if (threadIdx.x == 0) *reinterpret_cast<volatile int*>(err) = 5;
        return;
    }

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // (known to be uniform)
    const int kvh = blockIdx.x % a.kv_heads;
    const int n_rows = a.n * a.group;
    const int row0 = ((n_rows + QB - 1) / QB - 1 - (int)blockIdx.x / a.kv_heads) * QB;  // the longest rows first
    const int row_last = min(n_rows, row0 + QB) - 1;
    const Steps st = make_steps(a, a.start + row0 / a.group, a.start + row_last / a.group);
    const int per = (st.n + a.n_split - 1) / a.n_split;
    const int j0 = min(st.n, (int)blockIdx.y * per), j1 = min(st.n, j0 + per);
    int pa[TILES], pb[TILES];  // first and last position of each tile's rows
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        pa[t] = a.start + min(row0 + t * QT, row_last) / a.group;
        pb[t] = a.start + min(row0 + t * QT + QT - 1, row_last) / a.group;
    }
    const bool two = TILES == 2 && row0 + QT <= row_last;  // the second tile has rows
    auto cols = [&](int t, int j) { return t == 0 || two ? step_cols(a, st, j, pa[t], pb[t]) : Cols{0, 0}; };

    const int n_steps = j1 - j0;   // items of K, and of V, for the ring
    auto load = [&](bool v, int i) {   // f16, one thread
        const int s = Ring::at(v, i).stage, j = j0 + i, t0 = st.at(j);
        const CUtensorMap* map = j < st.n_first ? (v ? &tm_v_first : &tm_k_first) : (v ? &tm_v : &tm_k);
        mbar_expect_tx(&full[s], Y::STAGE);
#pragma unroll
        for (int b = 0; b < NB; b++) tma_load_3d(ring + s * Y::STAGE + b * (TK * 128), map, b * 64, t0, kvh, &full[s]);
    };
    if (warp == Y::LOAD_WARP && lane == 0) {
        ctl.dead = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&full[s], KIND == CACHE_Q4 ? 4 : 1);
            mbar_init(&empty[s], TILES);
        }
        for (int b = 0; b < 4; b++) {
            mbar_init(&p_ready[b], 4);
            mbar_init(&pv_done[b], 1);
            mbar_init(&drained[b], 1);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init(&s_full[t], 1);
            mbar_init(&s_read[t], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if constexpr (KIND == CACHE_F16)
            for (int k = 0, v = 0; k < min(n_steps, Ring::K) || v < min(n_steps, Ring::V);) {   // as many as there are stages
                const bool is_v = v < min(n_steps, Ring::V) && (k == min(n_steps, Ring::K) || Ring::next_is_v(k, v, n_steps));
                load(is_v, is_v ? v++ : k++);
            }
    }
    __syncwarp();
    if (warp == Y::MMA_WARP) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_slot)), "r"(Y::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // The queries, as f16 in the A operand's layout: row r of a tile, 16-byte chunk c of a 64-column block at r * 128 + ((c ^ (r & 7)) * 16).
    // Every warp takes batches of eight rows, lanes across head_dim, and has all of its loads on their way at once (the softmax warps alone, with one
    // batch ahead, took 9000 cycles for four latencies; a CTA of the 1792-row window prompt lives 45000).
    {
        constexpr int N = HD / 32, B = 8, BATCHES = QB / B, WARPS = Y::THREADS / 32, MINE = (BATCHES + WARPS - 1) / WARPS;
        float x[MINE][B][N];
#pragma unroll
        for (int k = 0; k < MINE; k++) {
            const int y0 = (warp + k * WARPS) * B;
            if (y0 >= QB) break;
            int i = min(row0 + y0, row_last) / a.group, g = min(row0 + y0, row_last) - i * a.group;
#pragma unroll
            for (int u = 0; u < B; u++) {
                const float* src = a.q + i * a.q_ld + (int64_t)(kvh * a.group + g) * HD + lane * N;
                if constexpr (N == 4) *reinterpret_cast<float4*>(x[k][u]) = *reinterpret_cast<const float4*>(src);
                else *reinterpret_cast<float2*>(x[k][u]) = *reinterpret_cast<const float2*>(src);
                if (row0 + y0 + u < row_last && ++g == a.group) { g = 0; i++; }   // (behind the last row: that row again)
            }
        }
#pragma unroll
        for (int k = 0; k < MINE; k++) {
            const int y0 = (warp + k * WARPS) * B;
            if (y0 >= QB) break;
            float c2 = 0.f;
#pragma unroll
            for (int u = 0; u < B; u++) {
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < N; e++) top = fmaxf(top, fabsf(x[k][u][e]));
                // the exponent of the largest magnitude, 2^e <= top < 2^(e+1); an infinite one keeps its factor (the row is
                // not finite and is computed again)
                int e = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23) - 127;
                e = e > 127 ? 0 : max(e, -100);
                const float up = row0 + y0 + u <= row_last ? __uint_as_float((uint32_t)(8 - e + 127) << 23) : 0.f;
                if (lane == u) c2 = rsqrtf((float)HD) * 1.4426950408889634f * __uint_as_float((uint32_t)(e - 8 + 127) << 23);
                __half2 h[N / 2], low[N / 2];   // x = h + low to 22 bits
#pragma unroll
                for (int v = 0; v < N / 2; v++) {
                    const float x0 = x[k][u][2 * v] * up, x1 = x[k][u][2 * v + 1] * up;
                    h[v] = __floats2half2_rn(x0, x1);
                    const float2 f = __half22float2(h[v]);
                    low[v] = __floats2half2_rn(x0 - f.x, x1 - f.y);
                }
                const int c = lane * N / 8;
                unsigned char* dst = q_s + y0 / QT * Y::Q_ROOM + (c >> 3) * (QT * 128) + (y0 % QT + u) * 128 + (((c & 7) ^ u) << 4) + (lane * N % 8) * 2;
                if constexpr (N == 4) {
                    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(h);
                    *reinterpret_cast<uint2*>(dst + Y::Q_HALF) = *reinterpret_cast<uint2*>(low);
                } else {
                    *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<uint32_t*>(h);
                    *reinterpret_cast<uint32_t*>(dst + Y::Q_HALF) = *reinterpret_cast<uint32_t*>(low);
                }
            }
            if (lane < B) c2_s[y0 + lane] = c2;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the MMA reads these through the async proxy
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = ctl.tmem_slot;

    // (one instruction for all warps of a warpgroup, whatever their roles)
    if (warp >= Y::MMA_WARP) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Y::OTHER_REGS));
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Y::SOFTMAX_REGS));
    if (warp >= Y::LOAD_WARP) {
        // ------------------------------- K and V steps into the ring -------------------------------------------------
        if constexpr (KIND == CACHE_F16) {
            if (warp == Y::LOAD_WARP && lane == 0) {
                int k = min(n_steps, Ring::K), v = min(n_steps, Ring::V);   // (the first are on their way)
                while (k < n_steps || v < n_steps) {
                    const bool is_v = Ring::next_is_v(k, v, n_steps);
                    const typename Ring::Slot slot = Ring::at(is_v, is_v ? v : k);
                    if (!mbar_wait(&empty[slot.stage], slot.parity ^ 1, dead, err)) break;
                    load(is_v, is_v ? v++ : k++);
                }
                for (int i = max(0, k - Ring::K); i < k; i++) mbar_drain(&full[Ring::at(false, i).stage], Ring::at(false, i).parity);   // no copy outlives the CTA
                for (int i = max(0, v - Ring::V); i < v; i++) mbar_drain(&full[Ring::at(true, i).stage], Ring::at(true, i).parity);
            } else if (warp > Y::LOAD_WARP && a.n_split == 1 && blockIdx.x + ahead < gridDim.x) {
                // The queries of the CTA that will have this one's place, into L2: the CTAs of a round start together, and memory is idle in
                // between (1792-row window prompt 68 us without, 66 with).
                const int next = blockIdx.x + ahead, kv_next = next % a.kv_heads, first = ((n_rows + QB - 1) / QB - 1 - next / a.kv_heads) * QB;
                for (int y = lane; y < QB && first + y < n_rows; y += 32) {
                    const int row = first + y;
                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.q + row / a.group * a.q_ld + (int64_t)(kv_next * a.group + row % a.group) * HD), "n"(HD * 4)
                                 : "memory");
                }
            }
        } else {
            // Four warps for K and four for V. A thread unpacks a quarter of a row: the same block of eight
            // values of every group (cache4.h), 32 rows a pass; the next AHEAD items of its warps are on their way.
            constexpr int G = HD / kQ4Group, ROWS = 32, PASSES = TK / ROWS, AHEAD = 2;
            const int x0 = (threadIdx.x - Y::LOAD_WARP * 32) & 127, quarter = x0 & 3, rr = x0 >> 2;
            const bool v = warp < Y::LOAD_WARP + 4;
            uint32_t w[AHEAD][PASSES][G];
            __half d[AHEAD][PASSES][G];
            const int64_t base = (int64_t)kvh * a.max_seq + rr;
            auto fetch = [&](int i, uint32_t (&w)[PASSES][G], __half (&d)[PASSES][G]) {
                const int j = j0 + i, t0 = st.at(j), end = (j < st.n_first ? min(a.sinks, a.start + a.n) : a.start + a.n) - t0 - rr;
                const uint8_t* codes = reinterpret_cast<const uint8_t*>(v ? a.v : a.k) + (base + t0) * (HD / 2) + quarter * (HD / 8);
                const __half* scales = (v ? a.v_scale : a.k_scale) + (base + t0) * G;
#pragma unroll
                for (int u = 0; u < PASSES; u++) {
                    if (u * ROWS < end) {
                        if constexpr (G == 4) {
                            *reinterpret_cast<uint4*>(w[u]) = *reinterpret_cast<const uint4*>(codes + u * ROWS * (HD / 2));
                            *reinterpret_cast<uint2*>(d[u]) = *reinterpret_cast<const uint2*>(scales + u * ROWS * G);
                        } else {
                            *reinterpret_cast<uint2*>(w[u]) = *reinterpret_cast<const uint2*>(codes + u * ROWS * (HD / 2));
                            *reinterpret_cast<uint32_t*>(d[u]) = *reinterpret_cast<const uint32_t*>(scales + u * ROWS * G);
                        }
                    } else {
#pragma unroll
                        for (int g = 0; g < G; g++) { w[u][g] = 0; d[u][g] = __ushort_as_half(0); }
                    }
                }
            };
            // (row rr + 32 u keeps rr's place in the swizzle pattern, so all passes store at constant offsets)
            uint32_t off[G];
#pragma unroll
            for (int g = 0; g < G; g++) {
                const int chunk = 4 * g + quarter;   // eight values 32 g + 8 quarter ...
                off[g] = (chunk >> 3) * (TK * 128) + rr * 128 + (((chunk & 7) ^ (rr & 7)) << 4);
            }
            bool ok = true;
            auto unpack = [&](int i, uint32_t (&w)[PASSES][G], __half (&d)[PASSES][G]) {
                const typename Ring::Slot slot = Ring::at(v, i);
                ok = ok && (!slot.used || warp_wait(&empty[slot.stage], slot.parity ^ 1, dead, err));
                if (!ok) return;
                unsigned char* dst = ring + slot.stage * Y::STAGE;
#pragma unroll
                for (int u = 0; u < PASSES; u++) {
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        const __half2 dd = __half2half2(d[u][g]);
                        __half2 h[4];
                        q4_pairs(w[u][g], h);
#pragma unroll
                        for (int e = 0; e < 4; e++) h[e] = __hmul2(h[e], dd);
                        *reinterpret_cast<uint4*>(dst + off[g] + u * ROWS * 128) = *reinterpret_cast<uint4*>(h);
                    }
                }
                if (i + AHEAD < n_steps) fetch(i + AHEAD, w, d);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[slot.stage]);
            };
#pragma unroll
            for (int u = 0; u < AHEAD; u++)
                if (u < n_steps) fetch(u, w[u], d[u]);
            for (int i = 0; i < n_steps && ok; i += AHEAD) {
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
                    if (i + u < n_steps) unpack(i + u, w[u], d[u]);
            }
        }
    } else if (warp >= Y::MMA_WARP) {
        // ------------------------------- MMA issuers -----------------------------------------------------------------
        // A warp for a tile's scores and one for its output products: a wait, a commit or the issue of eight MMAs costs 100 to 300 cycles each, and
        // one warp with all of a step's was busy for 1800 cycles, about as long as the softmax (512-row 4-bit chunk 153 us, with two warps 149; 8192-row prompt 278 and
        // 274).
        // The whole warp runs this and one thread issues: descriptors then live in uniform registers (from a branch of one
        // thread eight MMAs took 600 to 1400 cycles, longer than they run). Descriptors are a base plus a constant (the address is their low bits, in
        // units of 16 bytes), and a step that the tile sees whole goes through straight-line code.
        const int t = (warp - Y::MMA_WARP) % TILES;
        const bool leader = elect_one();
        // Steps that the tile sees whole: from the first that starts at its last row's window to the last that ends at its first row.
        const int whole0 = st.n_first + max(0, window_low(a, pb[t]) - st.l + TK - 1) / TK, whole1 = t == 0 || two ? st.n_first + (pa[t] + 1 - st.l) / TK : 0;
        auto cols_at = [&](int j) { return j >= whole0 && j < whole1 ? Cols{0, TK} : cols(t, j); };
        uint32_t done = 0;   // products issued
        bool ok = true;
        if (warp < Y::MMA_WARP + TILES) {
            const uint32_t idesc_s = (1u << 4) | ((uint32_t)(QT >> 4) << 24);   // | N / 8 << 17
            const uint64_t q_desc = desc_kmajor(smem_u32(q_s) + t * Y::Q_ROOM), k_desc = desc_kmajor(smem_u32(ring));
            for (int j = j0; j < j1 && ok; j++) {
                const typename Ring::Slot slot = Ring::at(false, j - j0);
                const uint32_t stage = slot.stage;
                const Cols c = cols_at(j);
                ok = warp_wait(&full[stage], slot.parity, dead, err);
                if (c.any() && done > 0) ok = ok && warp_wait(&s_read[t], (done - 1) & 1, dead, err);
                if (!ok) break;
                if (c.any()) {
                    tc_after();
                    const uint64_t kb = k_desc + (stage * Y::STAGE + (uint32_t)c.c0 * 128) / 16;
                    const uint32_t id = idesc_s | (uint32_t)((c.c1 - c.c0) >> 3) << 17, d = tmem + 2 * t * TK + c.c0;
#pragma unroll
                    for (int k = 0; k < HD / 16; k++)
                        if (leader) umma_ss(d, q_desc + ((k >> 2) * (QT * 128) + (k & 3) * 32) / 16, kb + ((k >> 2) * (TK * 128) + (k & 3) * 32) / 16, id, k > 0);
#pragma unroll
                    for (int k = 0; k < HD / 16; k++)   // and the low halves of the queries
                        if (leader) umma_ss(d, q_desc + (Y::Q_HALF + (k >> 2) * (QT * 128) + (k & 3) * 32) / 16, kb + ((k >> 2) * (TK * 128) + (k & 3) * 32) / 16, id, 1);
                    if (leader) umma_commit(&s_full[t]);
                    done++;
                }
                if (leader) umma_commit(&empty[stage]);
            }
        } else if (warp < Y::MMA_WARP + 2 * TILES) {
            const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(QT >> 4) << 24);
            const uint64_t v_desc = desc_mnmajor(smem_u32(ring), TK * 128);
            for (int j = j0; j < j1; j++) {   // the n-th product takes its weights from buffer n & 1
                const typename Ring::Slot slot = Ring::at(true, j - j0);
                const uint32_t stage = slot.stage, buf = done & 1;
                const Cols c = cols_at(j);
                ok = warp_wait(&full[stage], slot.parity, dead, err);
                if (c.any()) ok = ok && warp_wait(&p_ready[2 * t + buf], (done >> 1) & 1, dead, err);
                if (!ok) break;
                if (c.any()) {
                    tc_after();
                    const uint64_t vb = v_desc + stage * Y::STAGE / 16;
                    const uint32_t d = tmem + O_COL + t * HD, w = tmem + 2 * t * TK + TK + buf * (TK / 2);
                    if (c.c0 == 0 && c.c1 == TK) {
#pragma unroll
                        for (int k = 0; k < TK / 16; k++)
                            if (leader) umma_ts(d, w + k * 8, vb + k * 2048 / 16, idesc_o, k > 0 || done > 0);
                    } else {
                        for (int k = c.c0 / 16; k < c.c1 / 16; k++)
                            if (leader) umma_ts(d, w + k * 8, vb + k * 2048 / 16, idesc_o, k > c.c0 / 16 || done > 0);
                    }
                    if (leader) umma_commit(&pv_done[2 * t + buf]);
                    done++;
                }
                if (leader) umma_commit(&empty[stage]);
            }
        }
        if (leader) umma_commit(&drained[warp - Y::MMA_WARP]);   // no product outlives the CTA, whoever gave up
        mbar_drain(&drained[warp - Y::MMA_WARP], 0);
    } else {
        // ------------------------------- softmax: a thread owns a row ------------------------------------------------
        const int tile = warp >> 2, r = threadIdx.x & (QT - 1);   // the thread's tile and row
        const int row = min(row0 + tile * QT + r, row_last);
        const float c2 = c2_s[tile * QT + r];
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + lanes + 2 * tile * TK, o_addr = tmem + lanes + O_COL + tile * HD;
        const int p = a.start + row / a.group, low = window_low(a, p);
        // The row's weights are 2^(s c2 + shift), shift = kShift - m (FLT_MAX: nothing seen yet). It is the rounded shift that counts everywhere, in a
        // move's factor and in a record too: with scores beyond 2^23 it is not kShift - m any more.
        float shift = FLT_MAX, l = 0.f;
        uint32_t steps = 0;
        bool ok = true;
        const int warp_row = row0 + tile * QT + (warp & 3) * 32;   // the warp's first and last position
        const int wa = a.start + min(warp_row, row_last) / a.group, wb = a.start + min(warp_row + 31, row_last) / a.group;
        const int low_wb = window_low(a, wb);
        const uint64_t c2_2 = pack2(c2, c2);
        // One step; `whole`: every row of the warp sees all of it. One piece of code for both (with one for each, the rows' first steps waited for
        // instructions: 1792-row window prompt 73 us, so 68); what a row does not see, or nobody computed, weighs 2^-inf.
        auto step = [&](bool whole, int j, Cols now) {
            const uint32_t p_addr = s_addr + TK + (steps & 1) * (TK / 2);
            float x[TK];
            tmem_ld32_issue(s_addr, x);
            tmem_ld32_issue(s_addr + 32, x + 32);
            tmem_ld_wait();
            tmem_arrived(x);
            tmem_arrived(x + 32);
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_read[tile]);   // the next scores may come
            if (!whole) {
                // columns of the step that the row sees: below `to`, and from `from` on or below `first`
                const int t0 = st.at(j);
                const bool in_first = j < st.n_first;
                const int to = (in_first ? st.s : p + 1) - t0, from = (in_first ? 0 : low) - t0, first = (in_first ? 0 : a.sinks) - t0;
                auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
#pragma unroll
                for (int c = 0; c < TK; c += 32) {
                    const uint32_t sees = c < now.c0 || c >= now.c1 ? 0u : below(to - c) & (~below(from - c) | below(first - c));
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (!(sees >> e & 1)) x[c + e] = -INFINITY;
                }
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // four chains
#pragma unroll
            for (int e = 0; e < TK; e++) tops[e & 3] = fmaxf(tops[e & 3], x[e]);
            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * c2;
            const bool move = top + shift > kShift + kLag;
            if (__any_sync(0xffffffffu, move)) {
                const float shift_new = move ? kShift - top : shift, scale = ex2_approx(shift_new - shift);
                shift = shift_new;
                l *= scale;
                if (steps > 0) {
                    ok = warp_wait(&pv_done[2 * tile + ((steps - 1) & 1)], ((steps - 1) >> 1) & 1, dead, err);   // O is at rest
                    tc_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        float o[16];
                        tmem_ld16(o_addr + c, o);
                        uint32_t y[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) y[e] = __float_as_uint(o[e] * scale);
                        tmem_st16(o_addr + c, y);
                    }
                    tmem_st_wait();
                }
            }
            const uint64_t shift_2 = pack2(shift, shift);
            if (steps >= 2) ok = warp_wait(&pv_done[2 * tile + (steps & 1)], ((steps - 2) >> 1) & 1, dead, err) && ok;   // the weights two steps ago are used
            uint64_t sum[2] = {0, 0};   // two chains of two
#pragma unroll
            for (int c = 0; c < TK; c += 32) {
                uint32_t y[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    float w0, w1;
                    unpack2(fma2(pack2(x[c + 2 * e], x[c + 2 * e + 1]), c2_2, shift_2), w0, w1);
                    w0 = ex2_approx(w0);
                    w1 = ex2_approx(w1);
                    sum[e & 1] = add2(sum[e & 1], pack2(w0, w1));
                    const __half2 h = __floats2half2_rn(w0, w1);
                    y[e] = *reinterpret_cast<const uint32_t*>(&h);
                }
                tmem_st16(p_addr + c / 2, y);
            }
            float sum0, sum1;
            unpack2(add2(sum[0], sum[1]), sum0, sum1);
            l += sum0 + sum1;
            tmem_st_wait();
        };
        // steps that the warp sees whole: from the first that starts at its last row's window to the last that ends at its first row
        const int whole0 = st.n_first + max(0, low_wb - st.l + TK - 1) / TK, whole1 = tile == 0 || two ? st.n_first + (wa + 1 - st.l) / TK : 0;
        for (int j = j0; j < j1; j++) {
            const bool whole = j >= whole0 && j < whole1;
            const Cols now = whole ? Cols{0, TK} : cols(tile, j);
            if (!now.any()) continue;
            ok = warp_wait(&s_full[tile], steps & 1, dead, err);
            if (!ok) break;
            tc_after();
            step(whole, j, now);
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[2 * tile + (steps & 1)]);
            steps++;
            if (!ok) break;
        }
        if (ok && steps > 0) ok = warp_wait(&pv_done[2 * tile + ((steps - 1) & 1)], ((steps - 1) >> 1) & 1, dead, err);
        const bool live = row0 + tile * QT + r <= row_last;
        if (ok && __any_sync(0xffffffffu, live)) {
            tc_after();
            const int ii = row / a.group, head = kvh * a.group + row % a.group;
            const int64_t rec = ((int64_t)ii * a.heads + head) * a.n_split + blockIdx.y;
            // A row leaves through shared memory, from where one copy takes it out whole: the tile's scores are all computed, so its queries' room is
            // free. (Stored from registers by 16 lanes a row this was 5600 cycles of a CTA.)
            unsigned char *turn = q_s + tile * Y::Q_ROOM + (warp & 3) * (32 * Y::OUT_ROW), *mine = turn + lane * Y::OUT_ROW;
            const bool empty_row = p + 1 - low + min(a.sinks, low) == 0;
            const float inv = empty_row ? 0.f : 1.0f / l;
            float o_top = 0.f;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                float x[32];
                if (steps > 0) {
                    tmem_ld32(o_addr + c, x);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) x[e] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < 32; e++) max_abs_nan(o_top, x[e]);
                if (a.n_split > 1) {   // half a record at a time
                    unsigned char* dst = mine + c % (HD / 2) * 4;
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(dst + e * 4) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                    if ((c + 32) % (HD / 2) == 0) {
                        if (live) bulk_store(a.rec_o + rec * HD + c + 32 - HD / 2, mine, HD * 2);
                        __syncwarp();
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        __half2 h[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) h[u] = empty_row ? __half2half2(__ushort_as_half(0)) : __floats2half2_rn(x[e + 2 * u] * inv, x[e + 2 * u + 1] * inv);
                        *reinterpret_cast<uint4*>(mine + (c + e) * 2) = *reinterpret_cast<uint4*>(h);
                    }
                }
            }
            if (live && a.n_split > 1) a.rec_ml[rec] = make_float2(-shift, l);
            // Rows next to infinite or NaN cache contents that they do not see, again and one by one. So are those whose largest weight, 2^kShift when it was taken, has come out
            // as less than half of that or too large for f16: top is rounded before it is subtracted, the scores are not, and for scores beyond 2^23 the
            // difference is no longer small against 1. And rows that rounded weights have put beyond f16's largest value (see mean_f16).
            const bool beyond = a.n_split == 1 && o_top * inv >= kInfF16 && o_top <= FLT_MAX;
            __syncwarp();
            uint32_t bad = __ballot_sync(0xffffffffu, live && !empty_row && (row_is_suspect(l, o_top, shift) || (shift < FLT_MAX && l < 64.f) || beyond));
            if (bad && a.n_split > 1) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // (their records are there and may be replaced)
            __syncwarp();
            while (bad) {
                const int b = __ffs(bad) - 1;
                bad &= bad - 1;
                float o[HD / 32], sm, sl;
                slow_row<KIND, HD>(a, kvh, __shfl_sync(0xffffffffu, row, b), j0, j1, st, sm, sl, o);
                const int64_t rb = __shfl_sync(0xffffffffu, rec, b);
#pragma unroll
                for (int e = 0; e < HD / 32; e++) {
                    const int c = lane * (HD / 32) + e;
                    if (a.n_split > 1) a.rec_o[rb * HD + c] = o[e];
                    else *reinterpret_cast<__half*>(turn + b * Y::OUT_ROW + c * 2) = __float2half_rn(o[e] / sl);
                }
                if (a.n_split > 1 && lane == 0) a.rec_ml[rb] = make_float2(sm, sl);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (the row's own lane copies it)
                __syncwarp();
            }
            if (live && a.n_split == 1) bulk_store(reinterpret_cast<__half*>(a.out) + ii * a.out_ld + (int64_t)head * HD, mine, HD * 2);
        }
    }
    tc_before();
    __syncthreads();
    if (warp == Y::MMA_WARP) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Y::TMEM_COLS) : "memory");
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
    const int blocks = (a.n * a.group + Y::ROWS - 1) / Y::ROWS;
    kern<<<dim3((unsigned)(blocks * a.kv_heads), a.n_split), Y::THREADS, Y::SMEM, ctx->stream>>>(mk, mv, mkf, mvf, a, ctx->sm_count * (2 / Y::TILES), ctx->d_err);
    RLB_LAUNCH_CHECK();
    count_launch(ctx);
    return RLB_OK;
}

}  // namespace

// Splits of the positions: CTAs run in rounds over the SMs, and a CTA costs its share of the steps and about eight more (set-up,
// queries, masks, record or result). A split has at least eight steps.
int attn_long_tc_splits(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a) {
    if (ctx->attn_long_splits) return ctx->attn_long_splits;
    const int tiles = kind == CACHE_Q4 ? 2 : 1;
    const int64_t rows = tiles * QT, ctas = (int64_t)a.kv_heads * (((int64_t)a.n * a.group + rows - 1) / rows), slots = (int64_t)ctx->sm_count * (2 / tiles);
    const int64_t seen = std::min<int64_t>((int64_t)a.window + a.sinks + rows / a.group, (int64_t)a.start + a.n);
    const int64_t steps = (seen + TK - 1) / TK;
    int64_t best = 1, cost = INT64_MAX;
    for (int64_t s = 1; s <= std::max<int64_t>(1, std::min<int64_t>(steps / 8, std::min<int64_t>(64, record_limit(a)))); s++) {
        const int64_t c = ((ctas * s + slots - 1) / slots) * ((steps + s - 1) / s + 8);
        if (c < cost) { cost = c; best = s; }
    }
    return (int)best;
}

// 7 us (10 with the unpacking of 4-bit rows), the longer of the CTAs' steps, 1.15 us each (4 bits 1.3, with one tile 1.0; where the tensor cores are the
// bound up to a fifth more, which is not where the choice is close), and the reading of the cache, and for records 2.5 us and what it takes to write and read them.
double attn_long_tc_us(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a, int splits) {
    const int tiles = kind == CACHE_Q4 ? 2 : 1;
    const int64_t rows = tiles * QT, ctas = (int64_t)a.kv_heads * (((int64_t)a.n * a.group + rows - 1) / rows), slots = (int64_t)ctx->sm_count * (2 / tiles);
    const int64_t seen = std::min<int64_t>((int64_t)a.window + a.sinks + rows / a.group, (int64_t)a.start + a.n), steps = (seen + TK - 1) / TK;
    const double bytes = (double)seen * a.kv_heads * (kind == CACHE_Q4 ? a.hd + a.hd / 8 : a.hd * 4), step = kind == CACHE_F16 ? 1.15 : (int64_t)a.n * a.group > QT ? 1.3 : 1.0;
    const double records = splits > 1 ? 2.5 + 2.0 * a.n * a.heads * splits * (a.hd * 4 + 8) / 5e6 : 0;
    return (kind == CACHE_Q4 ? 10 : 7) + std::max(step * (double)((ctas * splits + slots - 1) / slots) * (double)((steps + splits - 1) / splits), bytes / 6.5e6) + records;
}

int launch_attn_long_tc(rlb_ctx* ctx, CacheKind kind, const AttnLongArgs& a) {
    if (kind == CACHE_F16) return a.hd == 128 ? launch<CACHE_F16, 128>(ctx, a) : launch<CACHE_F16, 64>(ctx, a);
    return a.hd == 128 ? launch<CACHE_Q4, 128>(ctx, a) : launch<CACHE_Q4, 64>(ctx, a);
}
