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

// The same for a 4-bit pool: a lane's dims lane + 32 i are one of each group, so a group's largest magnitude is a reduction
// over the warp; eight lanes put a word's nibbles together. pos0 NULL: one token, at position seq_lens[b] - 1.
struct Append4Params {
    uint8_t* pool;
    const int32_t* block_table;
    const int32_t* pos0;
    const int32_t* seq_lens;
    const void* k;
    const void* v;
    int64_t token_stride, seq_stride;
    int* err;
    int table_stride, batch, n_tokens, layer, n_layers, n_kv_heads, num_blocks, norm_k;
};

// The page of a position (block table entry pos / 128), or NULL with the error word set when the position lies outside the
// table's row or the entry outside the pool.
__device__ __forceinline__ uint8_t* page_of(uint8_t* pool, const int32_t* table_row, int table_stride, int num_blocks, int pos, int layer,
                                            int n_layers, int n_kv_heads, int h, size_t page_bytes, int* err) {
    const int e = pos / BLK;
    int block = -1;
    if (pos >= 0 && e < table_stride) block = table_row[e];
    if (block < 0 || block >= num_blocks) {
        atomicExch(err, ERR_BAD_BLOCK);
        return nullptr;
    }
    return pool + ((size_t(block) * n_layers + layer) * n_kv_heads + h) * page_bytes;
}

template <int DT>
__global__ void __launch_bounds__(128) kv4_append_kernel(const Append4Params p) {
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
    const int pos = p.pos0 ? p.pos0[b] + t : p.seq_lens[b] - 1;
    if (!p.pos0 && pos < 0) return;   // (an empty sequence has no current token)
    uint8_t* page = page_of(p.pool, p.block_table + size_t(b) * p.table_stride, p.table_stride, p.num_blocks, pos, p.layer, p.n_layers,
                            p.n_kv_heads, h, KV4_PAGE, p.err);
    if (!page) return;
    const int row = pos % BLK;
    float x[4];
    kv_row_load<DT>(is_v ? p.v : p.k, size_t(b) * p.seq_stride + size_t(t) * p.token_stride + size_t(h) * HD, !is_v && p.norm_k, lane, x);
    uint32_t word = 0;   // lane: word lane / 8 of group lane % 8 (lanes with lane % 8 < 4)
    __half scale = __ushort_as_half(0);   // lane g < 4: of group g
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[i] = Act<DT>::round(x[i]);
        const __half s = kv4_scale(warp_max_abs_nan(x[i]));
        uint32_t w = (uint32_t(kv4_code(x[i], __half2float(s))) & 15u) << (4 * kv4_nibble_of(lane & 7));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) w |= __shfl_xor_sync(0xffffffffu, w, o);
        if ((lane & 7) == i) word = w;
        if (lane == i) scale = s;
    }
    if ((lane & 7) < 4)
        *reinterpret_cast<uint32_t*>(page + is_v * KV4_SIDE + row * KV4_ROW + (lane & 7) * 16 + (lane >> 3) * 4) = word;
    if (lane < 4) reinterpret_cast<__half*>(page + 2 * KV4_SIDE)[row * 2 * KV4_GROUPS + is_v * KV4_GROUPS + lane] = scale;
}

// Rows of the cache back as activations: one warp per (sequence, token, kv head, K|V), a lane holds dims 4 lane .. 4 lane + 3.
struct ReadParams {
    uint8_t* pool;
    const int32_t* block_table;
    const int32_t* pos0;
    void* k;
    void* v;
    int64_t token_stride, seq_stride;
    size_t page_bytes;
    int* err;
    int table_stride, batch, n_tokens, layer, n_layers, n_kv_heads, num_blocks, kv_dtype, scale_bytes;
};

template <int DT>
__global__ void __launch_bounds__(128) kv_read_kernel(const ReadParams p) {
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
    const int pos = p.pos0[b] + t;
    const uint8_t* page = page_of(p.pool, p.block_table + size_t(b) * p.table_stride, p.table_stride, p.num_blocks, pos, p.layer,
                                  p.n_layers, p.n_kv_heads, h, p.page_bytes, p.err);
    if (!page) return;
    const int row = pos % BLK;
    uint2 out;
    if (p.kv_dtype == EMBLA_KV_16BIT) {
        out = reinterpret_cast<const uint2*>(page + is_v * (BLK * HD * 2) + row * HD * 2)[lane];
    } else {
        float x[4];
        if (p.kv_dtype == EMBLA_KV_INT4) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(page + is_v * KV4_SIDE + row * KV4_ROW)[lane >> 1];
            const float s = __half2float(reinterpret_cast<const __half*>(page + 2 * KV4_SIDE)[row * 2 * KV4_GROUPS + is_v * KV4_GROUPS + (lane >> 3)]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int n = kv4_nibble_of(4 * (lane & 1) + i);
                x[i] = float(int(w << (28 - 4 * n)) >> 28) * s;
            }
        } else {
            const char4 c = reinterpret_cast<const char4*>(page + is_v * CODE_BYTES + row * HD)[lane];
            const float s = load_scale(page + 2 * CODE_BYTES + is_v * BLK * p.scale_bytes, row, p.scale_bytes);
            x[0] = float(c.x) * s;
            x[1] = float(c.y) * s;
            x[2] = float(c.z) * s;
            x[3] = float(c.w) * s;
        }
        if (DT == EMBLA_F16) out = make_uint2(pack_h2(x[0], x[1]), pack_h2(x[2], x[3]));
        else {
            __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), c = __floats2bfloat162_rn(x[2], x[3]);
            out = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&c));
        }
    }
    uint16_t* dst = static_cast<uint16_t*>(is_v ? p.v : p.k) + size_t(b) * p.seq_stride + size_t(t) * p.token_stride + size_t(h) * HD;
    reinterpret_cast<uint2*>(dst)[lane] = out;
}

static EmblaStatus launch_append4(EmblaAttn* ctx, EmblaKVPool* pool, const EmblaKVView* view, const int32_t* pos0, int n_tokens,
                                  const void* k, const void* v, int64_t token_stride, int64_t seq_stride, int norm_k, cudaStream_t s) {
    Append4Params p;
    p.pool = pool->base;
    p.block_table = view->block_table_dev;
    p.pos0 = pos0;
    p.seq_lens = view->seq_lens_dev;
    p.k = k;
    p.v = v;
    p.token_stride = token_stride;
    p.seq_stride = seq_stride;
    p.err = ctx->err_dev;
    p.table_stride = view->table_stride;
    p.batch = view->batch;
    p.n_tokens = n_tokens;
    p.layer = view->layer;
    p.n_layers = pool->n_layers;
    p.n_kv_heads = pool->n_kv_heads;
    p.num_blocks = pool->num_blocks;
    p.norm_k = norm_k;
    const long warps = long(p.batch) * n_tokens * p.n_kv_heads * 2;
    if ((warps + 3) / 4 > 0x7fffffffL) EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_append: %d sequences x %d tokens are too many", p.batch, n_tokens);
    const dim3 grid(unsigned((warps + 3) / 4));
    if (ctx->cfg.act_dtype == EMBLA_BF16) EMBLA_CUDA_TRY(launch_kernel(ctx->pdl, kv4_append_kernel<EMBLA_BF16>, grid, dim3(128), 0, s, p));
    else EMBLA_CUDA_TRY(launch_kernel(ctx->pdl, kv4_append_kernel<EMBLA_F16>, grid, dim3(128), 0, s, p));
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
    ReadParams p;
    p.pool = pool->base;
    p.block_table = view->block_table_dev;
    p.pos0 = pos0_dev;
    p.k = k_dev;
    p.v = v_dev;
    p.token_stride = token_stride;
    p.seq_stride = seq_stride;
    p.page_bytes = pool->page_bytes;
    p.err = ctx->err_dev;
    p.table_stride = view->table_stride;
    p.batch = view->batch;
    p.n_tokens = n_tokens;
    p.layer = view->layer;
    p.n_layers = pool->n_layers;
    p.n_kv_heads = pool->n_kv_heads;
    p.num_blocks = pool->num_blocks;
    p.kv_dtype = pool->kv_dtype;
    p.scale_bytes = pool->scale_bytes;
    const long warps = long(p.batch) * n_tokens * p.n_kv_heads * 2;
    if ((warps + 3) / 4 > 0x7fffffffL) EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_read: %d sequences x %d tokens are too many", p.batch, n_tokens);
    const dim3 grid(unsigned((warps + 3) / 4));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (ctx->cfg.act_dtype == EMBLA_BF16) EMBLA_CUDA_TRY(launch_kernel(ctx->pdl, kv_read_kernel<EMBLA_BF16>, grid, dim3(128), 0, s, p));
    else EMBLA_CUDA_TRY(launch_kernel(ctx->pdl, kv_read_kernel<EMBLA_F16>, grid, dim3(128), 0, s, p));
    EMBLA_CUDA_TRY(cudaGetLastError());
    return EMBLA_OK;
}
