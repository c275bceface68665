// Attention over the 4-bit paged cache (EMBLA_KV_INT4): ReLU² of the full layers (prefill) and softmax of the
// sparse layers. First form: one CTA of 128 threads per query row; a thread takes one key of a page for the dots (fp32), then
// one head dim for the sum over the page's keys.
#include "kv4.cuh"

namespace embla {

struct Attend4Params {
    const uint8_t* pool;
    const int32_t* block_table;
    const int32_t* seq_lens;   // decode: keys of a sequence
    const int32_t* pos0;       // prefill: position of a sequence's first token; token t sees pos0 + t + 1 keys
    const uint32_t* idx;       // sparse: selected positions of sequences past 1152 keys
    const void* q;
    const void* g1;
    const void* g2;
    void* o;
    float* scores;
    int* err;
    int64_t q_token_stride, q_seq_stride, o_token_stride, o_seq_stride, scores_stride;
    int table_stride, layer, n_layers, n_kv_heads, num_blocks, G, prenormed, ng, softmax;
};

template <int DT>
__global__ void __launch_bounds__(128) kv4_attend_kernel(const Attend4Params p) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float q[HD], w[BLK], red[4];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int head = blockIdx.x, t = blockIdx.y, b = blockIdx.z, kvh = head / p.G;
    const int S = p.pos0 ? p.pos0[b] + t + 1 : p.seq_lens[b];
    const bool selecting = p.softmax && S > EMBLA_TOPK + EMBLA_RECENT;
    const int n = selecting ? EMBLA_TOPK + EMBLA_RECENT : max(S, 0);
    if (warp == 0) {
        const size_t off = size_t(b) * p.q_seq_stride + size_t(t) * p.q_token_stride + size_t(head) * HD;
        float x[4];
        kv_row_load<DT>(p.q, off, false, lane, x);
        if (!p.prenormed) kv4_query_norm<DT>(x, p.g1, p.g2, p.ng, lane);
        for (int i = 0; i < 4; i++) q[lane + 32 * i] = x[i];
    }
    __syncthreads();
    const float scale = rsqrtf(float(HD));
    float m = NEG_BIG, den = 0.0f, acc = 0.0f;
    for (int j0 = 0; j0 < n; j0 += BLK) {
        // this thread's key
        int pos = j0 + tid;
        bool valid = pos < n;
        if (selecting && valid) {
            const uint32_t r = p.idx[(size_t(b) * p.n_kv_heads + kvh) * (EMBLA_TOPK + EMBLA_RECENT) + pos];
            if (r >= uint32_t(S)) {
                atomicExch(p.err, ERR_BAD_BLOCK);
                valid = false;
            }
            pos = int(r);
        }
        const uint8_t* page = nullptr;
        if (valid) {
            const int e = pos / BLK, block = e < p.table_stride ? p.block_table[size_t(b) * p.table_stride + e] : -1;
            if (block < 0 || block >= p.num_blocks) {
                atomicExch(p.err, ERR_BAD_BLOCK);
                valid = false;
            } else {
                page = p.pool + ((size_t(block) * p.n_layers + p.layer) * p.n_kv_heads + kvh) * KV4_PAGE;
            }
        }
        float s = 0.0f;
        const int row = pos % BLK;
        if (valid) {
            const __half* sc = reinterpret_cast<const __half*>(page + 2 * KV4_SIDE) + row * 2 * KV4_GROUPS;
            for (int g = 0; g < KV4_GROUPS; g++) {
                float part = 0.0f;
                for (int c = 0; c < 4; c++) {
                    const uint32_t word = reinterpret_cast<const uint32_t*>(page + row * KV4_ROW)[g * 4 + c];
                    for (int d = 0; d < 8; d++) part = fmaf(q[g * 32 + c * 8 + d], float(int(word << (28 - 4 * kv4_nibble_of(d))) >> 28), part);
                }
                s = fmaf(part, __half2float(sc[g]), s);
            }
            if (p.scores) {   // max over the kv head's query heads: heads write one after another
                float* at = p.scores + (size_t(b) * p.n_kv_heads + kvh) * p.scores_stride + pos;
                if (s >= 0.0f) atomicMax(reinterpret_cast<int*>(at), __float_as_int(s));
                else atomicMin(reinterpret_cast<unsigned*>(at), __float_as_uint(s));
            }
        }
        s *= scale;
        if (p.softmax) {
            float mt = valid ? s : NEG_BIG;
            for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
            if (lane == 0) red[warp] = mt;
            __syncthreads();
            mt = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
            const float f = __expf(m - mt);
            den *= f;
            acc *= f;
            m = mt;
            s = valid ? __expf(s - m) : 0.0f;
        } else {
            s = valid ? fmaxf(s, 0.0f) : 0.0f;
            s *= s;
        }
        w[tid] = s;
        __syncthreads();
        // this thread's head dim
        const int word = tid >> 3, nib = kv4_nibble_of(tid & 7), g = tid >> 5;
        for (int k = 0; k < BLK && j0 + k < n; k++) {
            int ps = j0 + k;
            if (selecting) ps = int(p.idx[(size_t(b) * p.n_kv_heads + kvh) * (EMBLA_TOPK + EMBLA_RECENT) + ps]);
            const float wk = w[k];
            den += wk;
            if (wk == 0.0f) continue;   // (invalid keys among them)
            const int block = p.block_table[size_t(b) * p.table_stride + ps / BLK], r = ps % BLK;
            const uint8_t* pg = p.pool + ((size_t(block) * p.n_layers + p.layer) * p.n_kv_heads + kvh) * KV4_PAGE;
            const uint32_t c = reinterpret_cast<const uint32_t*>(pg + KV4_SIDE + r * KV4_ROW)[word];
            const float vs = __half2float(reinterpret_cast<const __half*>(pg + 2 * KV4_SIDE)[r * 2 * KV4_GROUPS + KV4_GROUPS + g]);
            acc = fmaf(wk, float(int(c << (28 - 4 * nib)) >> 28) * vs, acc);
        }
        __syncthreads();
    }
    const float total = p.softmax ? (den > 0.0f ? den : 1.0f) : sqrtf(float(HD)) + den;
    Act<DT>::store(p.o, size_t(b) * p.o_seq_stride + size_t(t) * p.o_token_stride + size_t(head) * HD + tid, acc / total);
}

static EmblaStatus launch_attend(EmblaAttn* ctx, Attend4Params& p, const EmblaKVPool* pool, const EmblaKVView* view, const EmblaQuery* q,
                                 int tokens, cudaStream_t s) {
    p.pool = pool->base;
    p.block_table = view->block_table_dev;
    p.seq_lens = view->seq_lens_dev;
    p.q = q->q_dev;
    p.g1 = q->g1_dev;
    p.g2 = q->g2_dev;
    p.err = ctx->err_dev;
    p.table_stride = view->table_stride;
    p.layer = view->layer;
    p.n_layers = pool->n_layers;
    p.n_kv_heads = pool->n_kv_heads;
    p.num_blocks = pool->num_blocks;
    p.G = ctx->cfg.n_q_heads / ctx->cfg.n_kv_heads;
    p.prenormed = q->prenormed;
    p.ng = q->ng;
    const dim3 grid(ctx->cfg.n_q_heads, tokens, view->batch);
    if (ctx->cfg.act_dtype == EMBLA_BF16) EMBLA_CUDA_TRY(launch_kernel(ctx->pdl, kv4_attend_kernel<EMBLA_BF16>, grid, dim3(128), 0, s, p));
    else EMBLA_CUDA_TRY(launch_kernel(ctx->pdl, kv4_attend_kernel<EMBLA_F16>, grid, dim3(128), 0, s, p));
    return EMBLA_OK;
}

EmblaStatus kv4_full_prefill(EmblaAttn* ctx, const EmblaKVPool* pool, const EmblaKVView* view, const int32_t* pos0, int n_tokens,
                             const EmblaQuery* q, int64_t q_token_stride, void* o_dev, int64_t o_token_stride, int64_t o_seq_stride,
                             cudaStream_t stream) {
    Attend4Params p = {};
    p.o = o_dev;
    p.pos0 = pos0;
    p.q_seq_stride = q->q_stride;
    p.q_token_stride = q_token_stride;
    p.o_seq_stride = o_seq_stride;
    p.o_token_stride = o_token_stride;
    return launch_attend(ctx, p, pool, view, q, n_tokens, stream);
}

}  // namespace embla
