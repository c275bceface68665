// Rows of the 4-bit cache (EMBLA_KV_INT4): 128 dims in four groups of 32, a fp16 scale each, codes -7 .. 7 as two's
// complement nibbles. A 32-bit word holds 8 consecutive dims, nibble n being dim (0, 2, 4, 6, 1, 3, 5, 7)[n]: the nibbles n and
// n + 4, which one mask takes out of the two halves of the word together, are then the neighbouring dims 2n and 2n + 1, so that
// widening a word gives fp16 pairs in dim order with no permutation.
#pragma once

#include "kv_row.cuh"

namespace embla {

__host__ __device__ constexpr int kv4_nibble_of(int d) { return (d >> 1) + 4 * (d & 1); }   // place of dim d (of 8) in its word

// The scale of a group whose largest magnitude is `top` (NaN or infinity: a NaN scale, so that what was not a number does not
// come back as one).
__device__ __forceinline__ __half kv4_scale(float top) {
    return top <= 3.4028234e38f ? __float2half_rn(fminf(__fdiv_rn(top, 7.0f), 65504.0f)) : __ushort_as_half(0x7fff);
}
// The code of x under the scale s, rint(x / s) clamped, as exact arithmetic gives it, from inv, the fp32 reciprocal of s. x and s
// have at most 11 significant bits, so x / s is either a half exactly or at least 2^-16 of its size away from one: x inv, off by
// 2^-23 of its size, lies on the right side of any half that x / s is not. If x / s is a half, x - code s is s / 2 either way
// (exact: code s has 14 bits), and the even code is taken.
__device__ __forceinline__ int kv4_code(float x, float s, float inv) {
    if (!(s > 0.0f)) return 0;
    float c = rintf(x * inv);
    const float rest = fmaf(-c, s, x);
    const int n = int(c);
    if (fabsf(rest) * 2.0f == s && (n & 1)) c += rest > 0.0f ? 1.0f : -1.0f;
    return int(fminf(fmaxf(c, -7.0f), 7.0f));
}
__device__ __forceinline__ float fmaxf_nan(float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); }

// The word of eight values under the scale of their group, whose largest magnitude is `top`; `scale` is set to it.
// Usually without a branch: top / 7 never is half-way between two normal fp16 values (seven times a 12-bit odd number has more
// than 11 bits), so the product with fp32 1 / 7 rounds to the same scale as the quotient; x inv + 1.5 2^23 rounds to an integer, the
// four codes of a half are put together as digits of base 16, and 8 is added to each digit and its sign bit flipped at the end.
// Quotients that are a half exactly (kv4_code), which every second warp meets among bf16 rows, are put right in a branch of their own
// (8 x 2048 tokens of 4 heads: bf16 17.1 us instead of 20.7). Subnormal scales and groups without one take the long way.
__device__ __forceinline__ uint32_t kv4_word(const float (&x)[8], float top, __half& scale) {
    constexpr float MAGIC = 12582912.0f;
    const float fast = top * (1.0f / 7.0f);
    scale = __float2half_rn(fast);
    const float s = __half2float(scale);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));   // (within an ulp)
    const bool slow = !(fast >= 6.2e-5f && fast <= 65000.0f);   // (normal fp16 with room to round either way; false for NaN)
    bool tie = false;
    float c[8];
#pragma unroll
    for (int d = 0; d < 8; d++) {
        c[d] = fmaf(x[d], inv, MAGIC) - MAGIC;
        tie |= fabsf(fmaf(-c[d], s, x[d])) == 0.5f * s;
    }
    if (tie) {
#pragma unroll
        for (int d = 0; d < 8; d++) {
            const float rest = fmaf(-c[d], s, x[d]);
            if (fabsf(rest) == 0.5f * s && (int(c[d]) & 1)) c[d] += rest > 0.0f ? 1.0f : -1.0f;
        }
    }
    const float lo = fmaf(fmaf(fmaf(c[6], 16.0f, c[4]), 16.0f, c[2]), 16.0f, c[0]);   // nibbles 3, 2, 1, 0
    const float hi = fmaf(fmaf(fmaf(c[7], 16.0f, c[5]), 16.0f, c[3]), 16.0f, c[1]);   // nibbles 7, 6, 5, 4
    const uint32_t l = __float_as_uint(lo + (MAGIC + 34952.0f)), h = __float_as_uint(hi + (MAGIC + 34952.0f));   // 0x8888
    uint32_t word = __byte_perm(l, h, 0x5410) ^ 0x88888888u;
    if (slow) {
        scale = kv4_scale(top);
        const float sf = __half2float(scale), si = sf > 0.0f ? __fdiv_rn(1.0f, sf) : 0.0f;
        word = 0;
#pragma unroll
        for (int d = 0; d < 8; d++) word |= (uint32_t(kv4_code(x[d], sf, si)) & 15u) << (4 * kv4_nibble_of(d));
    }
    return word;
}

// The query row of a head that comes raw: RMS norm over the head with `ng` gains, in the order of the other decode kernels
// (common.metal:30-41), rounded to the activation dtype. A lane holds dims lane + 32 i.
template <int DT>
__device__ __forceinline__ void kv4_query_norm(float (&x)[4], const void* g1, const void* g2, int ng, int lane) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) ss = __fadd_rn(ss, __fmul_rn(x[i], x[i]));
    float tot = 0.0f;
    for (int l = 0; l < 32; l++) tot = __fadd_rn(tot, __shfl_sync(0xffffffffu, ss, l));
    const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(tot, float(HD)), EPS32)));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float gn = r;
        if (ng >= 1) gn = __fmul_rn(gn, __fadd_rn(1.0f, Act<DT>::load(g1, lane + 32 * i)));
        if (ng >= 2) gn = __fmul_rn(gn, __fadd_rn(1.0f, Act<DT>::load(g2, lane + 32 * i)));
        x[i] = Act<DT>::round(__fmul_rn(x[i], gn));
    }
}

// Eight codes of a word -> four half2 (dims 0-1, 2-3, 4-5, 6-7), exactly: a nibble under the exponent of 1024 (low nibble of a
// byte, 1024 + code + 8 after the sign bit is flipped) or of 64 (high nibble: 64 + code + 8), minus that offset.
__device__ __forceinline__ uint32_t kv4_lop(uint32_t w, uint32_t mask, uint32_t flip) {
    uint32_t r;   // (w & mask) ^ flip, as one instruction
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(w), "r"(mask), "r"(flip));
    return r;
}
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
    __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
    __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
}
constexpr uint32_t KV4_LO_MASK = 0x000F000Fu, KV4_LO_FLIP = 0x64086408u, KV4_LO_OFF = 0x64086408u;   // half2(1032, 1032)
constexpr uint32_t KV4_HI_MASK = 0x00F000F0u, KV4_HI_FLIP = 0x54805480u, KV4_HI_OFF = 0x54805480u;   // half2(72, 72)
__device__ __forceinline__ void kv4_widen(uint32_t w, uint32_t (&h)[4]) {
    const uint32_t v = w >> 8;
    h[0] = h2_sub(kv4_lop(w, KV4_LO_MASK, KV4_LO_FLIP), KV4_LO_OFF);
    h[1] = h2_sub(kv4_lop(w, KV4_HI_MASK, KV4_HI_FLIP), KV4_HI_OFF);
    h[2] = h2_sub(kv4_lop(v, KV4_LO_MASK, KV4_LO_FLIP), KV4_LO_OFF);
    h[3] = h2_sub(kv4_lop(v, KV4_HI_MASK, KV4_HI_FLIP), KV4_HI_OFF);
}

}  // namespace embla
