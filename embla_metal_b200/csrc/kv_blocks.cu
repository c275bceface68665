// Copies of blocks inside a KV pool (embla_kv_copy_blocks): forking a sequence gives the new one its own copy of the last
// block's rows, moving blocks together frees the end of a pool. A page (one layer and kv head of a block) is a handful of
// arrays with a fixed number of bytes a position, so "the first r positions" are a leading piece of each.
//
// Bound by HBM: every byte is read and written once. 512 blocks of 442 KB take 71 us, 6.3 TB/s or 0.97 of the measured copy rate (a
// loop with one load in flight took 101); the last rows of 48 blocks (21 MB moved) 5.4 us.
#include "common.cuh"

namespace embla {

struct BlockSpan {
    int offset, row_bytes;   // where the array starts in a page, bytes a position
};
struct CopyParams {
    uint8_t* pool;
    const int32_t* src;
    const int32_t* dst;
    const int32_t* rows;
    size_t page_bytes, block_bytes;
    int* err;
    int num_blocks, pages, n_spans, ragged;   // pages: layers x kv heads of a block
    BlockSpan span[4];
};

// 16-byte loads in flight a thread: a 4-bit page (1152 words) is one batch of a CTA. 128 x 9, 384 x 3 and 320 x 4 measured the same.
constexpr int COPY_THREADS = 256, COPY_BATCH = 5;

__global__ void __launch_bounds__(COPY_THREADS) kv_copy_blocks_kernel(const __grid_constant__ CopyParams p) {
    const int i = int(blockIdx.x / unsigned(p.pages)), page = int(blockIdx.x % unsigned(p.pages));
    const int src = p.src[i], dst = p.dst[i];
    const int rows = p.rows ? max(0, min(BLK, p.rows[i])) : BLK;
    if (src < 0 || src >= p.num_blocks || dst < 0 || dst >= p.num_blocks) {
        if (threadIdx.x == 0) atomicExch(p.err, ERR_BAD_BLOCK);
        return;
    }
    const uint8_t* from = p.pool + size_t(src) * p.block_bytes + size_t(page) * p.page_bytes;
    uint8_t* to = p.pool + size_t(dst) * p.block_bytes + size_t(page) * p.page_bytes;
    // the pieces' whole 16-byte words, one piece after another
    int end[4];
#pragma unroll
    for (int k = 0; k < 4; k++) end[k] = (k ? end[k - 1] : 0) + (k < p.n_spans ? rows * p.span[k].row_bytes / 16 : 0);
    for (int base = int(threadIdx.x); base < end[3]; base += COPY_THREADS * COPY_BATCH) {
        uint4 v[COPY_BATCH];
        int at[COPY_BATCH];
#pragma unroll
        for (int u = 0; u < COPY_BATCH; u++) {
            const int w = base + u * COPY_THREADS;
            at[u] = p.span[0].offset + w * 16;
#pragma unroll
            for (int k = 1; k < 4; k++)
                if (w >= end[k - 1]) at[u] = p.span[k].offset + (w - end[k - 1]) * 16;
            if (w < end[3]) v[u] = __ldcs(reinterpret_cast<const uint4*>(from + at[u]));
        }
#pragma unroll
        for (int u = 0; u < COPY_BATCH; u++)
            if (base + u * COPY_THREADS < end[3]) __stcs(reinterpret_cast<uint4*>(to + at[u]), v[u]);
    }
    if (p.ragged) {   // int8 scales: an odd number of rows ends inside a word
        for (int k = 2; k < 4; k++) {
            const int bytes = rows * p.span[k].row_bytes, o = (bytes & ~15) + int(threadIdx.x) * 2;
            if (o < bytes) *reinterpret_cast<uint16_t*>(to + p.span[k].offset + o) = *reinterpret_cast<const uint16_t*>(from + p.span[k].offset + o);
        }
    }
}

}  // namespace embla

using namespace embla;

extern "C" EmblaStatus embla_kv_copy_blocks(EmblaAttn* ctx, EmblaKVPool* pool, const int32_t* src_dev, const int32_t* dst_dev,
                                            const int32_t* rows_dev, int32_t n, void* stream) {
    if (!ctx || !pool || (n > 0 && (!src_dev || !dst_dev))) EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_copy_blocks: null argument");
    if (n < 0) EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_copy_blocks: %d copies", n);
    EMBLA_CHECK_DEVICE("embla_kv_copy_blocks", ctx, pool);
    if (n == 0) return EMBLA_OK;
    CopyParams p = {};
    p.pool = pool->base;
    p.src = src_dev;
    p.dst = dst_dev;
    p.rows = rows_dev;
    p.page_bytes = pool->page_bytes;
    p.block_bytes = pool->block_bytes;
    p.err = ctx->err_dev;
    p.num_blocks = pool->num_blocks;
    p.pages = pool->n_layers * pool->n_kv_heads;
    if (pool->kv_dtype == EMBLA_KV_INT4) {
        p.n_spans = 3;
        p.span[0] = {0, KV4_ROW};
        p.span[1] = {KV4_SIDE, KV4_ROW};
        p.span[2] = {2 * KV4_SIDE, 2 * KV4_GROUPS * 2};
    } else if (pool->kv_dtype == EMBLA_KV_INT8) {
        p.n_spans = 4;
        p.ragged = 1;
        p.span[0] = {0, HD};
        p.span[1] = {CODE_BYTES, HD};
        p.span[2] = {2 * CODE_BYTES, pool->scale_bytes};
        p.span[3] = {2 * CODE_BYTES + BLK * pool->scale_bytes, pool->scale_bytes};
    } else {
        p.n_spans = 2;
        p.span[0] = {0, HD * 2};
        p.span[1] = {BLK * HD * 2, HD * 2};
    }
    const long ctas = long(n) * p.pages;
    if (ctas > 0x7fffffffL) EMBLA_FAIL(EMBLA_BAD_ARG, "embla_kv_copy_blocks: %d copies of %d pages are too many", n, p.pages);
    EMBLA_CUDA_TRY(launch_kernel(false, kv_copy_blocks_kernel, dim3(unsigned(ctas)), dim3(COPY_THREADS), 0, static_cast<cudaStream_t>(stream), p));
    EMBLA_CUDA_TRY(cudaGetLastError());
    return EMBLA_OK;
}
