// Copies of blocks inside a KV pool (embla_kv_copy_blocks): forking a sequence gives the new one its own copy of the last
// block's rows, moving blocks together frees the end of a pool. A page (one layer and kv head of a block) is a handful of
// arrays with a fixed number of bytes a position, so "the first r positions" are a leading piece of each.
//
// Bound by HBM: every byte is read and written once.
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
    int num_blocks, pages, n_spans;   // pages: layers x kv heads of a block
    BlockSpan span[4];
};

__global__ void __launch_bounds__(256) kv_copy_blocks_kernel(const CopyParams p) {
    const int i = int(blockIdx.x / unsigned(p.pages)), page = int(blockIdx.x % unsigned(p.pages));
    const int src = p.src[i], dst = p.dst[i];
    if (src < 0 || src >= p.num_blocks || dst < 0 || dst >= p.num_blocks) {
        if (threadIdx.x == 0) atomicExch(p.err, ERR_BAD_BLOCK);
        return;
    }
    const int rows = p.rows ? max(0, min(BLK, p.rows[i])) : BLK;
    const uint8_t* from = p.pool + size_t(src) * p.block_bytes + size_t(page) * p.page_bytes;
    uint8_t* to = p.pool + size_t(dst) * p.block_bytes + size_t(page) * p.page_bytes;
    for (int k = 0; k < p.n_spans; k++) {
        const int at = p.span[k].offset, bytes = rows * p.span[k].row_bytes, whole = bytes & ~15;
        for (int o = int(threadIdx.x) * 16; o < whole; o += 256 * 16)
            *reinterpret_cast<uint4*>(to + at + o) = *reinterpret_cast<const uint4*>(from + at + o);
        const int o = whole + int(threadIdx.x) * 2;   // (the scales of an odd number of int8 rows)
        if (o < bytes) *reinterpret_cast<uint16_t*>(to + at + o) = *reinterpret_cast<const uint16_t*>(from + at + o);
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
    EMBLA_CUDA_TRY(launch_kernel(false, kv_copy_blocks_kernel, dim3(unsigned(ctas)), dim3(256), 0, static_cast<cudaStream_t>(stream), p));
    EMBLA_CUDA_TRY(cudaGetLastError());
    return EMBLA_OK;
}
