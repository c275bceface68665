// Quantised KV append: the reference's kv_append / kv_append_b with write_row8
// (Sources/EmblaMetal/Kernels/attention.metal:113-140, prefill.metal:184-212, common.metal:74-84),
// writing into the paged pool. One warp per (sequence, token, kv head, K|V); a lane holds dims
// lane + 32 i like the reference. Every fp32 operation is an explicit round-to-nearest intrinsic in
// the order the CPU oracle uses, so codes and scales are bit-exact. A 16-bit pool (sparse layers that
// keep their own keys) takes the rows as they are, rounded to the activation dtype.
#include "kv4.cuh"

namespace embla {

struct AppendParams {
    uint8_t* pool;
    const int32_t* block_table;
    const int32_t* pos0;
    const void* k;
    const void* v;
    int64_t token_stride, seq_stride;
    size_t page_bytes;
    int table_stride, batch, n_tokens, layer, n_layers, n_kv_heads, scale_bytes, norm_k, kv16;
};

template <int DT>
__global__ void __launch_bounds__(128) kv_append_kernel(const AppendParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long warp = (long(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const long total = long(p.batch) * p.n_tokens * p.n_kv_heads * 2;
    if (warp >= total) return;
    const int is_v = int(warp & 1);
    const int h = int((warp >> 1) % p.n_kv_heads);
    const long bt = (warp >> 1) / p.n_kv_heads;
    const int t = int(bt % p.n_tokens), b = int(bt / p.n_tokens);
    const void* src = is_v ? p.v : p.k;
    const size_t off = size_t(b) * p.seq_stride + size_t(t) * p.token_stride + size_t(h) * HD;

    float x[4];
    kv_row_load<DT>(src, off, !is_v && p.norm_k, lane, x);
    const int pos = p.pos0[b] + t;
    const int block = p.block_table[size_t(b) * p.table_stride + pos / BLK];
    const int row = pos % BLK;
    uint8_t* page = p.pool + ((size_t(block) * p.n_layers + p.layer) * p.n_kv_heads + h) * p.page_bytes;
    if (p.kv16) {   // 16-bit pages: K rows [128][128], then V rows, in the activation dtype
        uint8_t* dst = page + (is_v ? BLK * HD * 2 : 0);
#pragma unroll
        for (int i = 0; i < 4; i++) Act<DT>::store(dst, size_t(row) * HD + lane + 32 * i, x[i]);
        return;
    }
    int code[4];
    float scale;
    kv_row_quantise<DT>(x, code, scale);
    int8_t* codes = reinterpret_cast<int8_t*>(page) + (is_v ? CODE_BYTES : 0) + row * HD;
#pragma unroll
    for (int i = 0; i < 4; i++) codes[lane + 32 * i] = int8_t(code[i]);
    if (lane == 0) {
        uint8_t* sc = page + 2 * CODE_BYTES + (is_v ? BLK * p.scale_bytes : 0);
        if (p.scale_bytes == 4) reinterpret_cast<float*>(sc)[row] = scale;
        else reinterpret_cast<__half*>(sc)[row] = __float2half_rn(scale);
    }
}

// ---- 4-bit pools, and reading rows back -------------------------------------------------------------------------------
// Half a warp takes a row: a lane holds 8 consecutive dims (16 bytes of activations, one word of codes), four lanes a scale
// group. A warp takes 2 x PASSES consecutive rows of one side (K or V), every load in flight before the first is used; lane i works
// out where row i lies, the others get it by shuffle. Bound by instructions (about 90 a row to quantise, 45 to read back), not by
// the bytes: 8 x 2048 tokens of 4 kv heads take 15.9 us to append (fp16, 17.1 bf16; 43 MB; 19.8 with the keys normed) and 11.5 us to
// read back, where a warp a row with two-byte loads took 93 us for the two.
// x / d for x < 2^30: (x mul) >> shift, mul = ceil(2^shift / d), shift = 30 + ceil(log2 d), whose error x (mul d - 2^shift) / (d 2^shift)
// is below 1 / d (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
struct Divisor {
    unsigned mul, shift;
    Divisor() = default;
    explicit Divisor(unsigned d) : shift(30) {
        while ((1ull << (shift - 30)) < d) shift++;
        mul = unsigned(((1ull << shift) + d - 1) / d);
    }
    __device__ __forceinline__ unsigned quotient(unsigned x) const { return unsigned((static_cast<unsigned long long>(x) * mul) >> shift); }
};
struct RowsParams {
    uint8_t* pool;
    const int32_t* block_table;
    const int32_t* pos0;       // NULL: one token, at position seq_lens[b] - 1
    const int32_t* seq_lens;
    void* k;                   // rows read (append) or written (read back)
    void* v;
    int64_t token_stride, seq_stride;
    size_t page_bytes;
    int* err;
    unsigned rows;             // of a side: batch x n_tokens x n_kv_heads, below 2^30
    Divisor by_heads, by_tokens;
    int table_stride, n_tokens, layer, n_layers, n_kv_heads, num_blocks, norm_k, kv_dtype, scale_bytes, vec;
};

// Where row i of a side lies: elements into k / v; page x 128 + row of the page (ROW_NOWHERE: no place, with the error word set).
constexpr unsigned ROW_NOWHERE = 0xffffffffu;
__device__ __forceinline__ long row_elements(const RowsParams& p, unsigned i, unsigned& b, unsigned& t, unsigned& h) {
    const unsigned bt = p.by_heads.quotient(i);
    h = i - bt * unsigned(p.n_kv_heads);
    b = p.by_tokens.quotient(bt);
    t = bt - b * unsigned(p.n_tokens);
    return long(b) * p.seq_stride + long(t) * p.token_stride + long(h) * HD;
}
__device__ __forceinline__ unsigned row_place(const RowsParams& p, unsigned b, unsigned t, unsigned h) {
    const int pos = p.pos0 ? p.pos0[b] + int(t) : p.seq_lens[b] - 1;
    if (!p.pos0 && pos < 0) return ROW_NOWHERE;   // (an empty sequence has no current token)
    int block = -1;
    if (pos >= 0 && pos / BLK < p.table_stride) block = p.block_table[size_t(b) * p.table_stride + pos / BLK];
    if (block < 0 || block >= p.num_blocks) {
        atomicExch(p.err, ERR_BAD_BLOCK);
        return ROW_NOWHERE;
    }
    return unsigned((long(block) * p.n_layers + p.layer) * p.n_kv_heads + long(h)) * BLK + unsigned(pos) % BLK;
}
__device__ __forceinline__ uint8_t* page_of(const RowsParams& p, unsigned place) { return p.pool + size_t(place / BLK) * p.page_bytes; }
template <int DT>
__device__ __forceinline__ float act_lo(uint32_t w) {
    return DT == EMBLA_BF16 ? __uint_as_float(w << 16) : __low2float(*reinterpret_cast<const __half2*>(&w));
}
template <int DT>
__device__ __forceinline__ float act_hi(uint32_t w) {
    return DT == EMBLA_BF16 ? __uint_as_float(w & 0xffff0000u) : __high2float(*reinterpret_cast<const __half2*>(&w));
}
template <int DT>
__device__ __forceinline__ uint32_t act_pack(float lo, float hi) {
    if (DT == EMBLA_F16) return pack_h2(lo, hi);
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}

constexpr int ROWS_WARPS = 4;

template <int DT, int PASSES, bool NORM>
__global__ void __launch_bounds__(ROWS_WARPS * 32) kv4_append_kernel(const __grid_constant__ RowsParams p) {
    // (keys to be normed: squares of a warp's rows, then their 32 partial sums a row, by the dims' order in the other append kernels)
    __shared__ float squares[NORM ? ROWS_WARPS : 1][NORM ? 2 * PASSES : 1][HD + 4];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = lane >> 4, col = lane & 15;
    const unsigned per = 2 * PASSES, groups = (p.rows + per - 1) / per;
    const unsigned unit = blockIdx.x * ROWS_WARPS + warp;
    if (unit >= 2 * groups) return;
    const bool is_v = unit >= groups;
    const unsigned first = (is_v ? unit - groups : unit) * per;
    const bool has = lane < int(per) && first + lane < p.rows;
    unsigned b = 0, t = 0, h = 0;
    const long elements = has ? row_elements(p, first + lane, b, t, h) : 0;
    uint4 x[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const long at = __shfl_sync(0xffffffffu, elements, 2 * i + half);
        const uint16_t* from = static_cast<const uint16_t*>(is_v ? p.v : p.k) + at + col * 8;
        x[i] = make_uint4(0, 0, 0, 0);
        if (first + 2 * i + half < p.rows) {
            if (p.vec) {
                x[i] = *reinterpret_cast<const uint4*>(from);
            } else {
                uint16_t e[8];
#pragma unroll
                for (int d = 0; d < 8; d++) e[d] = from[d];
                x[i] = make_uint4(e[0] | uint32_t(e[1]) << 16, e[2] | uint32_t(e[3]) << 16, e[4] | uint32_t(e[5]) << 16, e[6] | uint32_t(e[7]) << 16);
            }
        }
    }
    // (the lookups of the rows' pages run beside the loads of the rows)
    const unsigned mine = has ? row_place(p, b, t, h) : ROW_NOWHERE;
    if (NORM && !is_v) {
        // RMS norm without gains (common.metal:30-41): dims l, l + 32, l + 64, l + 96 into a partial sum each, then l = 0 .. 31
        float(*sq)[HD + 4] = squares[warp];
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            float* to = &sq[2 * i + half][col * 8];
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const float lo = act_lo<DT>(v[d]), hi = act_hi<DT>(v[d]);
                to[2 * d] = __fmul_rn(lo, lo);
                to[2 * d + 1] = __fmul_rn(hi, hi);
            }
        }
        __syncwarp();
        float part[2 * PASSES];
#pragma unroll
        for (int i = 0; i < 2 * PASSES; i++)
            part[i] = __fadd_rn(__fadd_rn(__fadd_rn(sq[i][lane], sq[i][lane + 32]), sq[i][lane + 64]), sq[i][lane + 96]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2 * PASSES; i++) sq[i][lane] = part[i];
        __syncwarp();
        float factor = 0.0f;
        if (lane < 2 * PASSES) {
            float tot = 0.0f;
#pragma unroll 8
            for (int l = 0; l < 32; l++) tot = __fadd_rn(tot, sq[lane][l]);
            factor = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(tot, float(HD)), EPS32)));
        }
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const float f = __shfl_sync(0xffffffffu, factor, 2 * i + half);
            uint32_t* v = &x[i].x;
#pragma unroll
            for (int d = 0; d < 4; d++) v[d] = act_pack<DT>(__fmul_rn(act_lo<DT>(v[d]), f), __fmul_rn(act_hi<DT>(v[d]), f));
        }
    }
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const unsigned place = __shfl_sync(0xffffffffu, mine, 2 * i + half);
        const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        // the group's largest magnitude: the types' bits without the sign are ordered as the magnitudes are, NaN on top
        uint32_t top = __vmaxu2(__vmaxu2(v[0] & 0x7fff7fffu, v[1] & 0x7fff7fffu), __vmaxu2(v[2] & 0x7fff7fffu, v[3] & 0x7fff7fffu));
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float xv[8];
#pragma unroll
        for (int d = 0; d < 4; d++) {
            xv[2 * d] = act_lo<DT>(v[d]);
            xv[2 * d + 1] = act_hi<DT>(v[d]);
        }
        __half sh;
        const uint32_t word = kv4_word(xv, fmaxf_nan(act_lo<DT>(top), act_hi<DT>(top)), sh);
        if (place == ROW_NOWHERE) continue;
        uint8_t* page = page_of(p, place);
        const int row = place % BLK;
        *reinterpret_cast<uint32_t*>(page + (is_v ? KV4_SIDE : 0) + row * KV4_ROW + col * 4) = word;
        if ((col & 3) == 0)
            reinterpret_cast<__half*>(page + 2 * KV4_SIDE)[row * 2 * KV4_GROUPS + (is_v ? KV4_GROUPS : 0) + (col >> 2)] = sh;
    }
}

template <int DT, int PASSES, bool INT4>
__global__ void __launch_bounds__(ROWS_WARPS * 32) kv_read_kernel(const __grid_constant__ RowsParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = lane >> 4, col = lane & 15;
    const unsigned per = 2 * PASSES, groups = (p.rows + per - 1) / per;
    const unsigned unit = blockIdx.x * ROWS_WARPS + warp;
    if (unit >= 2 * groups) return;
    const bool is_v = unit >= groups;
    const unsigned first = (is_v ? unit - groups : unit) * per;
    const bool has = lane < int(per) && first + lane < p.rows;
    unsigned b = 0, t = 0, h = 0;
    const long elements = has ? row_elements(p, first + lane, b, t, h) : 0;
    const unsigned mine = has ? row_place(p, b, t, h) : ROW_NOWHERE;
    unsigned place[PASSES];
    uint4 c[PASSES];   // the lane's 8 codes (or the row's values, 16-bit pools)
    float s[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        place[i] = __shfl_sync(0xffffffffu, mine, 2 * i + half);
        const uint8_t* page = page_of(p, place[i]);
        const int row = place[i] % BLK;
        c[i] = make_uint4(0, 0, 0, 0);
        s[i] = 0.0f;
        if (place[i] == ROW_NOWHERE) continue;
        if (INT4) {
            c[i].x = *reinterpret_cast<const uint32_t*>(page + (is_v ? KV4_SIDE : 0) + row * KV4_ROW + col * 4);
            s[i] = __half2float(reinterpret_cast<const __half*>(page + 2 * KV4_SIDE)[row * 2 * KV4_GROUPS + (is_v ? KV4_GROUPS : 0) + (col >> 2)]);
        } else if (p.kv_dtype == EMBLA_KV_INT8) {
            const uint2 t = *reinterpret_cast<const uint2*>(page + (is_v ? CODE_BYTES : 0) + row * HD + col * 8);
            c[i].x = t.x;
            c[i].y = t.y;
            s[i] = load_scale(page + 2 * CODE_BYTES + (is_v ? BLK * p.scale_bytes : 0), row, p.scale_bytes);
        } else {
            c[i] = *reinterpret_cast<const uint4*>(page + (is_v ? BLK * HD * 2 : 0) + row * HD * 2 + col * 16);
        }
    }
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const long at = __shfl_sync(0xffffffffu, elements, 2 * i + half);
        if (place[i] == ROW_NOWHERE) continue;
        uint4 out = c[i];
        if (p.kv_dtype != EMBLA_KV_16BIT) {
            uint32_t h[4];   // the codes as fp16 pairs, exactly
            if (INT4) {
                kv4_widen(c[i].x, h);
            } else {
                const uint32_t x0 = c[i].x ^ 0x80808080u, x1 = c[i].y ^ 0x80808080u;
                h[0] = h2_from_biased_bytes(x0, 0x4140);
                h[1] = h2_from_biased_bytes(x0, 0x4342);
                h[2] = h2_from_biased_bytes(x1, 0x4140);
                h[3] = h2_from_biased_bytes(x1, 0x4342);
            }
            uint32_t* to = &out.x;
            if (DT == EMBLA_F16 && INT4) {
                // (codes and scales are fp16: their fp16 product is the exact one rounded once, as below)
                const __half2 s2 = __float2half2_rn(s[i]);
#pragma unroll
                for (int d = 0; d < 4; d++) to[d] = h2_mul(h[d], *reinterpret_cast<const uint32_t*>(&s2));
            } else
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[d]));
                to[d] = act_pack<DT>(f.x * s[i], f.y * s[i]);
            }
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(is_v ? p.v : p.k) + at + col * 8) = out;
    }
}

// Rows a warp takes: eight (fewer lookups a row), or two while eight would leave an SM fewer than 32 warps (2048 tokens of 4 heads:
// 7.6 us with eight, 6.3 with four and less with two; 8 x 2048: 7 % less with eight than with four, 6 % less than with sixteen).
static int rows_passes(const EmblaAttn* ctx, unsigned rows) { return rows >= 128u * unsigned(ctx->sm_count) ? 4 : 1; }

static EmblaStatus rows_params(RowsParams& p, const char* fn, const EmblaKVPool* pool, const EmblaKVView* view, const int32_t* pos0, int n_tokens,
                               int64_t token_stride, int64_t seq_stride, const EmblaAttn* ctx) {
    const long rows = long(view->batch) * n_tokens * pool->n_kv_heads;
    if (rows > 0x3fffffffL) EMBLA_FAIL(EMBLA_BAD_ARG, "%s: %d sequences x %d tokens are too many", fn, view->batch, n_tokens);
    p.pool = pool->base;
    p.block_table = view->block_table_dev;
    p.pos0 = pos0;
    p.seq_lens = view->seq_lens_dev;
    p.token_stride = token_stride;
    p.seq_stride = seq_stride;
    p.page_bytes = pool->page_bytes;
    p.err = ctx->err_dev;
    p.rows = unsigned(rows);
    p.by_heads = Divisor(unsigned(pool->n_kv_heads));
    p.by_tokens = Divisor(unsigned(n_tokens));
    p.table_stride = view->table_stride;
    p.n_tokens = n_tokens;
    p.layer = view->layer;
    p.n_layers = pool->n_layers;
    p.n_kv_heads = pool->n_kv_heads;
    p.num_blocks = pool->num_blocks;
    p.kv_dtype = pool->kv_dtype;
    p.scale_bytes = pool->scale_bytes;
    return EMBLA_OK;
}
static dim3 rows_grid(unsigned rows, int passes) {
    const unsigned units = 2 * ((rows + 2 * passes - 1) / (2 * passes));
    return dim3((units + ROWS_WARPS - 1) / ROWS_WARPS);
}

static EmblaStatus launch_append4(EmblaAttn* ctx, EmblaKVPool* pool, const EmblaKVView* view, const int32_t* pos0, int n_tokens,
                                  const void* k, const void* v, int64_t token_stride, int64_t seq_stride, int norm_k, cudaStream_t s) {
    RowsParams p = {};
    if (EmblaStatus st = rows_params(p, "embla_kv_append", pool, view, pos0, n_tokens, token_stride, seq_stride, ctx)) return st;
    p.k = const_cast<void*>(k);
    p.v = const_cast<void*>(v);
    p.norm_k = norm_k;
    p.vec = token_stride % 8 == 0 && seq_stride % 8 == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0;
    const int passes = rows_passes(ctx, p.rows);
    const bool bf = ctx->cfg.act_dtype == EMBLA_BF16;
#define EMBLA_A4(DT, P) (norm_k ? launch_kernel(ctx->pdl, kv4_append_kernel<DT, P, true>, rows_grid(p.rows, P), dim3(ROWS_WARPS * 32), 0, s, p) \
                                : launch_kernel(ctx->pdl, kv4_append_kernel<DT, P, false>, rows_grid(p.rows, P), dim3(ROWS_WARPS * 32), 0, s, p))
    if (passes == 4) EMBLA_CUDA_TRY(bf ? EMBLA_A4(EMBLA_BF16, 4) : EMBLA_A4(EMBLA_F16, 4));
    else EMBLA_CUDA_TRY(bf ? EMBLA_A4(EMBLA_BF16, 1) : EMBLA_A4(EMBLA_F16, 1));
#undef EMBLA_A4
    EMBLA_CUDA_TRY(cudaGetLastError());
    return EMBLA_OK;
}

EmblaStatus kv4_append_token(EmblaAttn* ctx, EmblaKVPool* pool, const EmblaKVView* view, const void* k_dev, const void* v_dev,
                             int64_t kv_stride, int norm_k, cudaStream_t stream) {
    return launch_append4(ctx, pool, view, nullptr, 1, k_dev, v_dev, kv_stride, kv_stride, norm_k, stream);
}

}  // namespace embla

using namespace embla;

extern "C" EmblaStatus embla_kv_append(EmblaAttn* ctx, EmblaKVPool* pool, const EmblaKVView* view,
                                       const int32_t* pos0_dev, int32_t n_tokens,
                                       const void* k_dev, const void* v_dev, int64_t token_stride, int64_t seq_stride,
                                       int32_t norm_k, void* stream) {
    if (!ctx || !pool || !view || !pos0_dev || !k_dev || !v_dev) EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_append: null argument");
    EMBLA_CHECK_DEVICE("embla_kv_append", ctx, pool);
    if (view->layer < 0 || view->layer >= pool->n_layers)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_append: layer %d outside the pool's %d", view->layer, pool->n_layers);
    if (view->batch <= 0 || n_tokens <= 0 || !view->block_table_dev)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_append: batch %d, n_tokens %d", view->batch, n_tokens);
    if (pool->n_kv_heads != ctx->cfg.n_kv_heads)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_append: pool has %d kv heads, context %d", pool->n_kv_heads, ctx->cfg.n_kv_heads);
    if (pool->kv_dtype == EMBLA_KV_INT4)
        return launch_append4(ctx, pool, view, pos0_dev, n_tokens, k_dev, v_dev, token_stride, seq_stride, norm_k,
                              static_cast<cudaStream_t>(stream));
    AppendParams p;
    p.pool = pool->base;
    p.block_table = view->block_table_dev;
    p.pos0 = pos0_dev;
    p.k = k_dev;
    p.v = v_dev;
    p.token_stride = token_stride;
    p.seq_stride = seq_stride;
    p.page_bytes = pool->page_bytes;
    p.table_stride = view->table_stride;
    p.batch = view->batch;
    p.n_tokens = n_tokens;
    p.layer = view->layer;
    p.n_layers = pool->n_layers;
    p.n_kv_heads = pool->n_kv_heads;
    p.scale_bytes = pool->scale_bytes;
    p.norm_k = norm_k;
    p.kv16 = pool->kv_dtype == EMBLA_KV_16BIT;
    const long warps = long(p.batch) * n_tokens * p.n_kv_heads * 2;
    const unsigned blocks = unsigned((warps + 3) / 4);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (ctx->cfg.act_dtype == EMBLA_BF16) EMBLA_CUDA_TRY(launch_kernel(ctx->pdl, kv_append_kernel<EMBLA_BF16>, dim3(blocks), dim3(128), 0, s, p));
    else EMBLA_CUDA_TRY(launch_kernel(ctx->pdl, kv_append_kernel<EMBLA_F16>, dim3(blocks), dim3(128), 0, s, p));
    EMBLA_CUDA_TRY(cudaGetLastError());
    return EMBLA_OK;
}

extern "C" EmblaStatus embla_kv_read(EmblaAttn* ctx, const EmblaKVPool* pool, const EmblaKVView* view, const int32_t* pos0_dev,
                                     int32_t n_tokens, void* k_dev, void* v_dev, int64_t token_stride, int64_t seq_stride,
                                     void* stream) {
    if (!ctx || !pool || !view || !pos0_dev || !k_dev || !v_dev) EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_read: null argument");
    EMBLA_CHECK_DEVICE("embla_kv_read", ctx, pool);
    if (view->layer < 0 || view->layer >= pool->n_layers)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_read: layer %d outside the pool's %d", view->layer, pool->n_layers);
    if (view->batch <= 0 || n_tokens <= 0 || !view->block_table_dev)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_read: batch %d, n_tokens %d", view->batch, n_tokens);
    if (pool->n_kv_heads != ctx->cfg.n_kv_heads)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_read: pool has %d kv heads, context %d", pool->n_kv_heads, ctx->cfg.n_kv_heads);
    if (token_stride % 8 || seq_stride % 8 || reinterpret_cast<uintptr_t>(k_dev) % 16 || reinterpret_cast<uintptr_t>(v_dev) % 16)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_read: strides must be multiples of 8 elements and the outputs 16-byte aligned");
    RowsParams p = {};
    if (EmblaStatus st = rows_params(p, "embla_kv_read", pool, view, pos0_dev, n_tokens, token_stride, seq_stride, ctx)) return st;
    p.k = k_dev;
    p.v = v_dev;
    const int passes = rows_passes(ctx, p.rows);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf = ctx->cfg.act_dtype == EMBLA_BF16;
    const bool int4 = pool->kv_dtype == EMBLA_KV_INT4;
#define EMBLA_RD(DT, P) (int4 ? launch_kernel(ctx->pdl, kv_read_kernel<DT, P, true>, rows_grid(p.rows, P), dim3(ROWS_WARPS * 32), 0, s, p) \
                              : launch_kernel(ctx->pdl, kv_read_kernel<DT, P, false>, rows_grid(p.rows, P), dim3(ROWS_WARPS * 32), 0, s, p))
    if (passes == 4) EMBLA_CUDA_TRY(bf ? EMBLA_RD(EMBLA_BF16, 4) : EMBLA_RD(EMBLA_F16, 4));
    else EMBLA_CUDA_TRY(bf ? EMBLA_RD(EMBLA_BF16, 1) : EMBLA_RD(EMBLA_F16, 1));
#undef EMBLA_RD
    EMBLA_CUDA_TRY(cudaGetLastError());
    return EMBLA_OK;
}
