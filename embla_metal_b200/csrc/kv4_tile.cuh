// The arithmetic of a 16-key tile of the 4-bit cache on a warp's tensor-core tiles (m16n8k16, fp16 operands, fp32 sums), for up to
// 8 query heads of a kv head. Rows of 64 code bytes lie in shared memory as TMA puts them there: two rows a 128-byte line, 16-byte
// chunk c of line l at c ^ (l % 8), which is conflict-free for every access below.
//
//   S^T = K Q^T   A = 16 keys x 16 dims. A row's chunk g is its group g: ldmatrix hands lane (r, t) the word of key r that holds
//                 dims 8t .. 8t + 7 of the group, which widens to the A registers of two products with no permutation. The
//                 products of a group are summed apart (fp32), times the key's scale of the group into S. The ALU pipe (two
//                 instructions a clock and SM) is what a decode runs out of first, so a word costs it one shift and four logic
//                 operations and no more: a nibble stays where it is, its sign bit flipped, as the fp16 subnormal
//                 (code + 8) 2^-24 (low nibble of a byte) or (code + 8) 2^-20 (high nibble), exact in the product; the queries
//                 of the low nibbles' dims carry the missing 2^4. The constant part, 8 x the sum of the query over the group,
//                 is the accumulator's start value, negated. What that costs, against 64 bits: 2^-20.8 of sum |q| |k| for rows of
//                 even size (bf16 queries 2^-24), at most 2^-18.5 of max |q| sum |k| for any (queries that span 2^24, keys of
//                 one code a group): the offset's terms are up to 15 max |q| in size, whatever the key.
//   O^T = V^T P^T A = 16 dims x 16 keys. The transposing ldmatrix, on 16-bit elements of four codes, hands lane (r, t) the
//                 element r of keys 2t and 2t + 1 side by side: widened, its nibbles are A registers (a dim, two keys). The
//                 value's scale of the group is multiplied into P (a B register a group), the codes stay exact. (As subnormals
//                 the codes would save the subtraction here too, but the tensor pipe adds products below the largest by their
//                 exponents, a subnormal's as if it were 2^-14: ten bits of the sums of values were lost.)
#pragma once

#include "kv4.cuh"

namespace embla {

// byte of 16-byte chunk `chunk` (group) of row `row` in a side
__device__ __forceinline__ int kv4_at(int row, int chunk) { return (row >> 1) * 128 + (((((row & 1) << 2) | chunk) ^ ((row >> 1) & 7)) << 4); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix4_trans(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float relu_nan(float x) {   // max(x, 0), NaN of NaN
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(x));
    return r;
}
// 2^(e - 127) for a biased exponent 1 .. 254
__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float(uint32_t(e) << 23); }

constexpr float KV4_SUBNORMAL = 1.0f / 1048576.0f;   // 2^-20: S comes out of the products scaled by it

// D = A B + C with C apart from D, fp16 operands, fp32 sums (not volatile: the products of two tiles may be interleaved)
__device__ __forceinline__ void mma_16816_c(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                            const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// The queries of a kv head in shared memory: rows scaled by a power of two that brings their largest element into [1, 2), so that fp16
// holds bf16 rows of any size, elements below 2^-14 of the largest to 2^-25 of it; and what goes with them.
struct Kv4Queries {
    __half q[8][HD];
    int expo[8];                  // biased exponent of the power of two; 0: no such head
};

// Dims in the order of the B registers: of every 8, those in low nibbles (0, 1, 4, 5), then those in high ones (2, 3, 6, 7), so that
// the two registers of a product come out of one load side by side.
__device__ __forceinline__ int kv4_q_column(int d) { return (d & ~6) | ((d & 4) >> 1) | ((d & 2) << 1); }

// One warp, one head: its row as it lies (zeros for a head the kv head does not have); then head norm if asked, scaled and stored.
template <int DT>
__device__ __forceinline__ void kv4_load_query(float (&x)[4], bool has, const void* q, size_t off, int lane) {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = has ? Act<DT>::load(q, off + lane + 32 * i) : 0.0f;
}
template <int DT>
__device__ __forceinline__ void kv4_stage_query(Kv4Queries& sq, int hh, bool has, float (&x)[4], bool prenormed, const void* g1, const void* g2,
                                                int ng, int lane) {
    if (has && !prenormed) kv4_query_norm<DT>(x, g1, g2, ng, lane);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    const int e = min(max(int(top >> 23), 1), 253);
    const float down = pow2_biased(254 - e);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half h = __float2half_rn(x[i] * down);
        // dims 0, 1, 4, 5 of every 8 lie in low nibbles: 16 x (exact)
        sq.q[hh][kv4_q_column(lane) + 32 * i] = (lane & 2) ? h : __hmul(h, __float2half_rn(16.0f));
    }
    if (lane == 0) sq.expo[hh] = has ? e : 0;
}

// A lane's share of the queries: B registers of head r = lane / 4, the products' start values of heads
// 2t, 2t + 1 (t = lane % 4).
struct Kv4Frag {
    uint32_t b[KV4_GROUPS][4];
    float start[KV4_GROUPS][4];
    __device__ __forceinline__ void load(const Kv4Queries& sq, int lane) {
        const int r = lane >> 2, t = lane & 3;
#pragma unroll
        for (int g = 0; g < KV4_GROUPS; g++) {
            const uint4 v = *reinterpret_cast<const uint4*>(&sq.q[r][32 * g + 8 * t]);
            b[g][0] = v.x;
            b[g][1] = v.y;
            b[g][2] = v.z;
            b[g][3] = v.w;
            // -8 x the sum over the group, in the products' own way: rows of -8 2^-24 and -8 2^-20
            const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma_16816_c(start[g], 0x80088008u, 0x80088008u, 0x80088008u, 0x80088008u, b[g][0], b[g][1], zero);
            mma_16816_c(start[g], 0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u, b[g][2], b[g][3], start[g]);
        }
    }
};

// This lane's ldmatrix address in a tile whose row 0 is a multiple of 16 rows into the side: groups 0 and 1; ^ 32 for 2 and 3.
__device__ __forceinline__ int kv4_lane_at(int lane) { return kv4_at((((lane >> 3) & 1) << 3) | (lane & 7), lane >> 4); }

// The scale rows of a lane's keys r and r + 8 of a tile (`sc`: its rows [16][8]): K groups in x, y, V groups in z, w.
struct Kv4Scales {
    uint4 k0, k1;
    __device__ __forceinline__ void load(const uint8_t* sc, int lane) {
        k0 = *reinterpret_cast<const uint4*>(sc + (lane >> 2) * 16);
        k1 = *reinterpret_cast<const uint4*>(sc + ((lane >> 2) + 8) * 16);
    }
    // some value scale of 2 or more (one test of a bit), and of 8 or more or NaN: its product with a weight of 2^13 could leave fp16
    __device__ __forceinline__ bool large() const { return ((k0.z | k0.w | k1.z | k1.w) & 0x40004000u) != 0; }
    __device__ __forceinline__ bool wide() const {
        const uint32_t top = __vmaxu2(__vmaxu2(k0.z, k0.w), __vmaxu2(k1.z, k1.w));
        return (top & 0xffffu) >= 0x4800u || (top >> 16) >= 0x4800u;
    }
    // keys of the tile from `lim` on: their value scales may be anything, NaN included, and become zero
    __device__ __forceinline__ void mask(int lane, int lim) {
        if ((lane >> 2) >= lim) k0.z = k0.w = 0;
        if ((lane >> 2) + 8 >= lim) k1.z = k1.w = 0;
    }
};

// S of 16 keys: s[0], s[1] key r, heads 2t, 2t + 1; s[2], s[3] key r + 8. `kaddr`: shared address of the tile's key rows plus
// kv4_lane_at.
__device__ __forceinline__ void kv4_tile_scores(uint32_t kaddr, const Kv4Scales& sc, const Kv4Frag& f, float (&s)[4]) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
        uint32_t w[4];
        ldmatrix4(w, kaddr ^ (j * 32));
        const float2 ks0 = __half22float2(*reinterpret_cast<const __half2*>(j ? &sc.k0.y : &sc.k0.x));
        const float2 ks1 = __half22float2(*reinterpret_cast<const __half2*>(j ? &sc.k1.y : &sc.k1.x));
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int g = 2 * j + h;
            const uint32_t lo = w[2 * h], hi = w[2 * h + 1];   // keys r and r + 8
            const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
            float a[4];
            // dims 0, 1 and 4, 5 of the lane's eight, then 2, 3 and 6, 7
            mma_16816_c(a, kv4_lop(lo, KV4_LO_MASK, 0x00080008u), kv4_lop(hi, KV4_LO_MASK, 0x00080008u), kv4_lop(lo8, KV4_LO_MASK, 0x00080008u),
                        kv4_lop(hi8, KV4_LO_MASK, 0x00080008u), f.b[g][0], f.b[g][1], f.start[g]);
            mma_16816_c(a, kv4_lop(lo, KV4_HI_MASK, 0x00800080u), kv4_lop(hi, KV4_HI_MASK, 0x00800080u), kv4_lop(lo8, KV4_HI_MASK, 0x00800080u),
                        kv4_lop(hi8, KV4_HI_MASK, 0x00800080u), f.b[g][2], f.b[g][3], a);
            const float x0 = h ? ks0.y : ks0.x, x1 = h ? ks1.y : ks1.x;
            if (g == 0) {
                s[0] = a[0] * x0;
                s[1] = a[1] * x0;
                s[2] = a[2] * x1;
                s[3] = a[3] * x1;
            } else {
                s[0] = fmaf(a[0], x0, s[0]);
                s[1] = fmaf(a[1], x0, s[1]);
                s[2] = fmaf(a[2], x1, s[2]);
                s[3] = fmaf(a[3], x1, s[3]);
            }
        }
    }
}

// O^T += V^T P^T for the tile: w[0], w[1] the weights of key r for heads 2t, 2t + 1, w[2], w[3] of key r + 8. A weight times
// the value's scale is rounded to fp16 once (2^-11, fp32 before) where the output is fp16; where it is bf16, whose own rounding
// is eight times larger, the weight and the product are rounded both, which saves 22 instructions a tile (64 x 32768 keys: 218 us
// instead of 230). An 8 x 8 transpose makes it the B register of head r, keys 2t,
// 2t + 1. Accumulator tile 2g + p holds, in [0], [1], dim 32 g + 8 (r / 2) + (r % 2) + 4 p of heads 2t, 2t + 1, in [2], [3]
// that dim + 2.
template <int DT>
__device__ __forceinline__ void kv4_tile_values(uint32_t vaddr, const Kv4Scales& sc, const float (&w)[4], float (&O)[8][4]) {
    const uint32_t pw0 = pack_h2(w[0], w[1]), pw1 = pack_h2(w[2], w[3]);   // (bf16)
#pragma unroll
    for (int j = 0; j < 2; j++) {
        uint32_t x[4];
        ldmatrix4_trans(x, vaddr ^ (j * 32));
        const __half2 s0 = *reinterpret_cast<const __half2*>(j ? &sc.k0.w : &sc.k0.z), s1 = *reinterpret_cast<const __half2*>(j ? &sc.k1.w : &sc.k1.z);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int g = 2 * j + h;
            uint32_t b0, b1;
            if (DT == EMBLA_BF16) {
                const __half2 x0 = h ? __high2half2(s0) : __low2half2(s0), x1 = h ? __high2half2(s1) : __low2half2(s1);
                b0 = h2_mul(pw0, *reinterpret_cast<const uint32_t*>(&x0));
                b1 = h2_mul(pw1, *reinterpret_cast<const uint32_t*>(&x1));
            } else {
                const float x0 = h ? __high2float(s0) : __low2float(s0), x1 = h ? __high2float(s1) : __low2float(s1);
                b0 = pack_h2(w[0] * x0, w[1] * x0);
                b1 = pack_h2(w[2] * x1, w[3] * x1);
            }
            b0 = movmatrix4_trans(b0);
            b1 = movmatrix4_trans(b1);
            uint32_t lo[4], hi[4];
            kv4_widen(x[2 * h], lo);
            kv4_widen(x[2 * h + 1], hi);
            mma_16816_c(O[2 * g], lo[0], lo[1], hi[0], hi[1], b0, b1, O[2 * g]);
            mma_16816_c(O[2 * g + 1], lo[2], lo[3], hi[2], hi[3], b0, b1, O[2 * g + 1]);
        }
    }
}

// The same where a weight times a scale may leave fp16 (Kv4Scales::wide): the product in fp32, as the sum of two bf16 numbers (2^-17), so
// that groups of any size keep their bits beside one another; two products a tile, codes widened to bf16 (64 x 32768 keys with every value
// scale above 8: 318 us, without 228 in fp16 and 216 in bf16; a warp that kept its weights below 1/2 instead left groups of 0.01
// beside one of 100 a few bits).
__device__ __forceinline__ void mma_16816_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four codes of a word's low nibbles (of the bytes 0 and 2) -> bf16 pairs: 128 + code + 8 under the exponent of 128, minus 136
__device__ __forceinline__ uint32_t kv4_low_bf16(uint32_t w) {
    const uint32_t x = (w & KV4_LO_MASK) ^ 0x43084308u, off = 0x43084308u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&off));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void kv4_tile_values_wide(uint32_t vaddr, const Kv4Scales& sc, const float (&w)[4], float (&O)[8][4]) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
        uint32_t x[4];
        ldmatrix4_trans(x, vaddr ^ (j * 32));
        const float2 s0 = __half22float2(*reinterpret_cast<const __half2*>(j ? &sc.k0.w : &sc.k0.z));
        const float2 s1 = __half22float2(*reinterpret_cast<const __half2*>(j ? &sc.k1.w : &sc.k1.z));
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int g = 2 * j + h;
            float b[4] = {w[0] * (h ? s0.y : s0.x), w[1] * (h ? s0.y : s0.x), w[2] * (h ? s1.y : s1.x), w[3] * (h ? s1.y : s1.x)};
#pragma unroll
            for (int part = 0; part < 2; part++) {
                uint32_t b0 = pack_bf16(b[0], b[1]), b1 = pack_bf16(b[2], b[3]);
                b[0] -= __uint_as_float(b0 << 16);
                b[1] -= __uint_as_float(b0 & 0xffff0000u);
                b[2] -= __uint_as_float(b1 << 16);
                b[3] -= __uint_as_float(b1 & 0xffff0000u);
                b0 = movmatrix4_trans(b0);
                b1 = movmatrix4_trans(b1);
                const uint32_t lo = x[2 * h], hi = x[2 * h + 1];
                mma_16816_bf16(O[2 * g], kv4_low_bf16(lo), kv4_low_bf16(lo >> 4), kv4_low_bf16(hi), kv4_low_bf16(hi >> 4), b0, b1);
                mma_16816_bf16(O[2 * g + 1], kv4_low_bf16(lo >> 8), kv4_low_bf16(lo >> 12), kv4_low_bf16(hi >> 8), kv4_low_bf16(hi >> 12), b0, b1);
            }
        }
    }
}
__device__ __forceinline__ int kv4_dim_of(int tile, int r) { return 32 * (tile >> 1) + 8 * (r >> 1) + (r & 1) + 4 * (tile & 1); }

}  // namespace embla
