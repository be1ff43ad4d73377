// The 4-bit cache format.
//
// Per K or V row (one K/V head, one position, hd = 64 or 128 values) and per group of 32 neighbouring values there is one
// f16 scale d and 32 codes u of 4 bits, -7 <= u <= 7; the value is d * u. With m the group's largest magnitude (at most
// 65504), d = f16(bf16(m * f32(1/7))) and u = x / d rounded to the nearest integer (ties to even), clamped to 7. The
// detour over bf16 leaves d eight significant bits; u has three, so d * u has at most eleven: every value that the cache
// holds IS an f16 number, and the f16 tensor-core operands made from it carry no rounding of their own. The price is at
// most 2^-9 of the step. A group of zeros (or of magnitudes below the smallest scale) has d = 0; a group holding a NaN
// has d = NaN, so all of it reads back as NaN; infinities count as +-65504.
//
// Codes are stored as nibbles u + 8 in 32-bit words of eight neighbouring values. Inside a word, nibble j < 4 holds value
// 2j and nibble j + 4 value 2j + 1, so one shift and one mask give a pair of neighbours in the two halves of a register.
// The words of a row are ordered [block of eight inside the group][group]: word (e % 32) / 8 * (hd / 32) + e / 32 holds
// value e. Four threads that read a quarter of the row each then hold the same share of every group, which is how a
// tensor-core fragment wants its contraction index (four threads share one) with the group's scale factored out.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

constexpr int kQ4Group = 32;

#ifdef __CUDACC__
// The pair of values 2j, 2j + 1 of a word, without their scale: exact small integers.
__device__ __forceinline__ __half2 q4_pair(uint32_t word, int j) {
    const uint32_t t = ((word >> (4 * j)) & 0x000F000Fu) | 0x64006400u;  // 1024 + nibble: the nibble is the mantissa's low end
    const uint32_t bias = 0x64086408u;                                   // 1032
    return __hsub2(*reinterpret_cast<const __half2*>(&t), *reinterpret_cast<const __half2*>(&bias));
}
__host__ __device__ __forceinline__ int q4_word(int e, int groups) { return (e % kQ4Group) / 8 * groups + e / kQ4Group; }

// The four pairs of a word: the nibbles in the upper half of a byte are taken in place, as 1024 + 16 u.
__device__ __forceinline__ void q4_pairs(uint32_t word, __half2 (&h)[4]) {
    const uint32_t bias = 0x64086408u, sixteenth = 0x2C002C00u, high_bias = 0xD480D480u;  // 1032, 1/16, -72 = -(1024 / 16 + 8)
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const uint32_t w = b ? word >> 8 : word;
        uint32_t lo, hi;   // (w & mask) | 0x64006400
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(lo) : "r"(w), "r"(0x000F000Fu), "r"(0x64006400u));
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(hi) : "r"(w), "r"(0x00F000F0u), "r"(0x64006400u));
        h[2 * b] = __hsub2(*reinterpret_cast<const __half2*>(&lo), *reinterpret_cast<const __half2*>(&bias));
        h[2 * b + 1] = __hfma2(*reinterpret_cast<const __half2*>(&hi), *reinterpret_cast<const __half2*>(&sixteenth), *reinterpret_cast<const __half2*>(&high_bias));
    }
}

// Scale of a group whose largest magnitude is m.
__device__ __forceinline__ __half q4_scale(float m) {
    return __float2half_rn(__bfloat162float(__float2bfloat16_rn(__fmul_rn(fminf(m, 65504.f), 1.0f / 7.0f))));
}
// Eight values into a word: the nibbles 8 + rint(x / d), clamped. x * (1 / d), with an approximate reciprocal, is within 2e-6 of x / d below 8, so it rounds to the
// same integer unless it lies next to a half; only then is the quotient itself needed. (A correctly rounded division for every value is most of
// the arithmetic of an append, which is then bound by it.) Adding 1.5 * 2^23 + 8 rounds to the nearest even and leaves the nibble in the lowest bits
// of the sum; what stands above them is the same for all and is taken off the word once. (A rounding and a conversion to an integer for each value
// kept that unit busy for 64 % of an append, at the same 40 us for 1792 rows and their reading back: latency beside 76 % of the issue slots now.)
__device__ __forceinline__ uint32_t q4_pack(const float (&x)[8], float d) {
    if (!(d > 0.f)) return 0x88888888u;
    constexpr float kRound = 12582920.f;
    constexpr uint32_t kBits = 0x4B400000u;   // of 1.5 * 2^23
    const float inv = __fdividef(1.0f, d);
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float t = fminf(fmaxf(x[e] * inv, -7.f), 7.f);
        float y = t + kRound;
        if (fabsf(t - (y - kRound)) > 0.49999f) y = fminf(fmaxf(__fdiv_rn(x[e], d), -7.f), 7.f) + kRound;
        const int shift = 4 * ((e >> 1) + (e & 1) * 4);
        w += (__float_as_uint(y) - kBits) << shift;
    }
    return w;
}
#endif
