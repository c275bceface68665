// Decode attention of sparse layers over a 4-bit paged cache (EMBLA_KV_INT4): softmax over every key of a sequence with at most
// 1152, else over the rows idx[kv head][0..1151] that embla_select_keys wrote. No counterpart in the reference, whose cache is
// int8 (attn_sparse8 / attn_sparse_short, attention.metal:448-645; sparse8_decode.cu).
//
// A row is 144 bytes in nine 16-byte pieces at an address that two dependent lookups give (selected position, its block), so this
// is a matter of latency and of rows in flight. Each warp works alone: it looks up all its rows, then takes them 32 at a time, the
// copies (cp.async) of two groups in flight, two 16-key tiles of a group at once on the tensor-core tiles of kv4_tile.cuh. Its
// softmax keeps a reference score that moves (the sums with it) only when a weight passes 2^13. Up to eight CTAs a (sequence, kv
// head), as a thread-block cluster, when there are few of them.
//
// 64 sequences of 32768 keys, 4 kv heads: 27 to 29 us for 42 MB of rows (56 MB read: a row's scales are 16 bytes of the 64 that the HBM
// gives), 4 sequences of 9000: 9.0 to 10.3 us, of which 6 are launch, lookups and one row's way here. 31 instructions a row, 39 % of the
// issue slots; the same number of rows side by side instead of scattered take 17.6 us.
#include "attn16_common.cuh"
#include "kv4_tile.cuh"

namespace embla {

constexpr int KS_WARPS = 4, KS_STAGES = 2, KS_ROWS = 32;   // (three stages leave room for three CTAs an SM, not four)
constexpr int KS_STAGE = KS_ROWS * (2 * KV4_ROW + 4 * KV4_GROUPS);   // a group's rows: K codes, V codes, scales: 4608 bytes
constexpr int KS_SUM = HD + 1, KS_PART = HD + 4;                     // floats of a row of sums: in shared memory, between CTAs
constexpr int KS_MAX_CLUSTER = 8;
// largest weight, and the log2 of the one a moved reference gives the row's largest score (large value scales: kv4_tile_values_wide)
constexpr float KS_LIMIT = 8192.0f, KS_TARGET = 10.0f;
constexpr int KS_MAX_GROUPS = (EMBLA_TOPK + EMBLA_RECENT) / KS_ROWS / KS_WARPS;   // of a warp, in a CTA that has all rows to itself
constexpr uint32_t KS_NOWHERE = 0xffffffffu;
constexpr float KS_NONE = -1e30f;                                    // a reference before any key

struct Kv4SparseParams {
    const uint8_t* pool;
    const int32_t* block_table;
    const uint32_t* idx;
    const int32_t* seq_lens;
    const void* q;
    const void* g1;
    const void* g2;
    void* o;
    KernelCtl ctl;
    int64_t q_stride, o_stride;
    int table_stride, layer, n_layers, n_kv_heads, num_blocks, G, prenormed, ng, nsplit;
};

constexpr size_t ks_queries_at() { return size_t(KS_WARPS) * KS_STAGES * KS_STAGE; }
constexpr size_t ks_where_at() { return ks_queries_at() + sizeof(Kv4Queries); }
constexpr size_t ks_inbox_at() { return ks_where_at() + size_t(KS_WARPS) * KS_MAX_GROUPS * KS_ROWS * 4; }
constexpr int ks_inbox_rows(int ranges, int G) { return ranges * ((G + ranges - 1) / ranges); }
constexpr size_t ks_smem(int ranges, int G) { return 1024 + ks_inbox_at() + (ranges > 1 ? size_t(ks_inbox_rows(ranges, G)) * KS_PART * 4 : 0); }
static_assert(KS_WARPS * 8 * (KS_SUM + 2) * 4 <= KS_WARPS * KS_STAGES * KS_STAGE, "the warps' sums lie over their stages");

// 16 bytes (zeros if not `valid`) into shared memory; on a miss the L2 fetches the 64 bytes around them and not the 128 that it
// fetches by itself, since a row's neighbour is no more likely to be selected than any (64 x 32768 keys: 28.8 us instead of 31.0).
__device__ __forceinline__ void copy16(void* dst, const void* src, bool valid) {
    const uint32_t bytes = valid ? 16u : 0u;
    asm volatile("cp.async.cg.shared.global.L2::64B [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float ks_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <int DT, bool CL>
__global__ void __launch_bounds__(KS_WARPS * 32, 4) kv4_sparse_kernel(const __grid_constant__ Kv4SparseParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Kv4Queries& sq = *reinterpret_cast<Kv4Queries*>(smem + ks_queries_at());
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    trace_first(p.ctl.trace, 0);
    if (CL) cluster_arrive();   // (every CTA of the cluster has started before any writes into another's shared memory)
    const int S = max(0, p.seq_lens[b]);   // (read ahead of the wait: nothing on the GPU writes the sequence lengths)
    pdl_wait();
    pdl_launch_dependents();
    trace_first(p.ctl.trace, 1);
    const bool selecting = S > EMBLA_TOPK + EMBLA_RECENT && p.idx != nullptr;
    const int count = min(S, EMBLA_TOPK + EMBLA_RECENT);   // (no list given: no sequence is longer, says the caller)
    // the groups of 32 rows, dealt to the warps of the CTAs in turn
    const int groups = (count + KS_ROWS - 1) / KS_ROWS;
    const uint32_t* idx = p.idx + (size_t(b) * p.n_kv_heads + kvh) * (EMBLA_TOPK + EMBLA_RECENT);
    const int32_t* table = p.block_table + size_t(b) * p.table_stride;
    uint8_t* stage0 = smem + warp * (KS_STAGES * KS_STAGE);
    const int step = p.nsplit * KS_WARPS, first = split * KS_WARPS + warp;

    // Where the rows of all the warp's groups lie, as (page x 128 + row of the page), or KS_NOWHERE (behind the last one, or outside
    // the pool): the selected positions' loads in flight together, then those of the blocks, so that the chain of lookups is
    // walked once and not every group.
    uint32_t* where = reinterpret_cast<uint32_t*>(smem + ks_where_at()) + warp * (KS_MAX_GROUPS * KS_ROWS);
    {
        uint32_t pos[KS_MAX_GROUPS];
        int block[KS_MAX_GROUPS];
#pragma unroll
        for (int i = 0; i < KS_MAX_GROUPS; i++) {
            const int j = (first + i * step) * KS_ROWS + lane;
            pos[i] = 0xffffffffu;
            if (j < count) pos[i] = selecting ? idx[j] : uint32_t(j);
        }
#pragma unroll
        for (int i = 0; i < KS_MAX_GROUPS; i++) {
            block[i] = -1;
            if (pos[i] < uint32_t(S) && int(pos[i] / BLK) < p.table_stride) block[i] = table[pos[i] / BLK];
        }
#pragma unroll
        for (int i = 0; i < KS_MAX_GROUPS; i++) {
            uint32_t at = KS_NOWHERE;
            if (block[i] >= 0 && block[i] < p.num_blocks)
                at = uint32_t((long(block[i]) * p.n_layers + p.layer) * p.n_kv_heads + kvh) * BLK + pos[i] % BLK;
            else if ((first + i * step) * KS_ROWS + lane < count) atomicExch(p.ctl.err, ERR_BAD_BLOCK);
            where[i * KS_ROWS + lane] = at;
        }
        __syncwarp();
    }
    // The copies of the warp's group i into its stage; rows that are nowhere become zeros. Every call makes one copy group.
    auto request = [&](int i) {
        if (first + i * step < groups) {
            uint8_t* dst = stage0 + i % KS_STAGES * KS_STAGE;
            const uint32_t* at = where + i * KS_ROWS;
#pragma unroll
            for (int it = 0; it < 4; it++) {
                const int row = it * 8 + (lane >> 2), ch = lane & 3;
                const uint32_t a = at[row];
                const uint8_t* src = p.pool + (a == KS_NOWHERE ? 0 : size_t(a / BLK) * KV4_PAGE + (a % BLK) * KV4_ROW + ch * 16);
                copy16(dst + kv4_at(row, ch), src, a != KS_NOWHERE);
                copy16(dst + KS_ROWS * KV4_ROW + kv4_at(row, ch), src + KV4_SIDE, a != KS_NOWHERE);
            }
            const uint32_t a = at[lane];
            const uint8_t* src = p.pool + (a == KS_NOWHERE ? 0 : size_t(a / BLK) * KV4_PAGE + 2 * KV4_SIDE + (a % BLK) * 16);
            copy16(dst + 2 * KS_ROWS * KV4_ROW + lane * 16, src, a != KS_NOWHERE);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the first two groups' rows on their way, then the queries
#pragma unroll
    for (int i = 0; i < KS_STAGES - 1; i++) request(i);
#pragma unroll
    for (int i = 0; i < 8 / KS_WARPS; i++) {
        const int hh = warp + i * KS_WARPS;
        float x[4];
        kv4_load_query<DT>(x, hh < p.G, p.q, size_t(b) * p.q_stride + size_t(kvh * p.G + hh) * HD, lane);
        kv4_stage_query<DT>(sq, hh, hh < p.G, x, p.prenormed != 0, p.g1, p.g2, p.ng, lane);
    }
    __syncthreads();

    const int r = lane >> 2, t = lane & 3;
    Kv4Frag frag;
    frag.load(sq, lane);
    // scores in units of log2(e) / sqrt(128) x the query's power of two x 2^20. (Queries above 2^60 as if they were that large: the scores stay
    // inside fp32, and any two of them that differ already leave the smaller one no weight.)
    const float u0 = pow2_biased(min(max(sq.expo[2 * t], 1), 187)) * (1.4426950408889634f * 0.08838834764831845f / KV4_SUBNORMAL);
    const float u1 = pow2_biased(min(max(sq.expo[2 * t + 1], 1), 187)) * (1.4426950408889634f * 0.08838834764831845f / KV4_SUBNORMAL);
    float O[8][4];
#pragma unroll
    for (int i = 0; i < 8; i++) O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.0f;
    float l0 = 0.0f, l1 = 0.0f, m0 = KS_NONE, m1 = KS_NONE;   // sums of weights, reference scores of heads 2t, 2t + 1
#pragma unroll 1
    for (int i = 0; first + i * step < groups; i++) {
        request(i + KS_STAGES - 1);
        const unsigned ok = __ballot_sync(0xffffffffu, where[i * KS_ROWS + lane] != KS_NOWHERE);
        asm volatile("cp.async.wait_group %0;" ::"n"(KS_STAGES - 1) : "memory");
        __syncwarp();
        const uint8_t* rows = stage0 + i % KS_STAGES * KS_STAGE;
        const uint32_t kaddr = smem_u32(rows) + kv4_lane_at(lane);
        float s[2][4];
        Kv4Scales sc[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            sc[k].load(rows + 2 * KS_ROWS * KV4_ROW + k * 256, lane);
            kv4_tile_scores(kaddr + k * 16 * KV4_ROW, sc[k], frag, s[k]);
        }
        float w[2][4], top = 0.0f;
        bool flagged = false;
        auto weigh = [&]() {
            top = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const bool k0 = (ok >> (16 * k + r)) & 1, k1 = (ok >> (16 * k + r + 8)) & 1;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    // (a NaN score stays one; the product is rounded before the reference is taken off, as the reference was when it was taken: what a
                    // fused operation would keep of a score of 2^31 is more than exp2 can take)
                    w[k][e] = (e < 2 ? k0 : k1) ? ks_exp2(__fsub_rn(__fmul_rn(s[k][e], (e & 1) ? u1 : u0), (e & 1) ? m1 : m0)) : 0.0f;
                    top = fmaxf(top, w[k][e]);
                }
            }
        };
        weigh();
        flagged = sc[0].large() || sc[1].large();
        bool wide = false;
        if (__any_sync(0xffffffffu, flagged)) wide = __any_sync(0xffffffffu, sc[0].wide() || sc[1].wide());
        if (__any_sync(0xffffffffu, top > KS_LIMIT)) {
            // new references, no lower than the old: the group's largest score of a head weighs 2^target or less
            float t0 = KS_NONE, t1 = KS_NONE;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const bool k0 = (ok >> (16 * k + r)) & 1, k1 = (ok >> (16 * k + r + 8)) & 1;
                if (k0) t0 = fmaxf(t0, __fmul_rn(s[k][0], u0)), t1 = fmaxf(t1, __fmul_rn(s[k][1], u1));
                if (k1) t0 = fmaxf(t0, __fmul_rn(s[k][2], u0)), t1 = fmaxf(t1, __fmul_rn(s[k][3], u1));
            }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
                t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
            }
            const float n0 = fmaxf(m0, __fsub_ru(t0, KS_TARGET)), n1 = fmaxf(m1, __fsub_ru(t1, KS_TARGET));   // (no lower, whatever the scores' size)
            const float c0 = ks_exp2(m0 - n0), c1 = ks_exp2(m1 - n1);
            m0 = n0;
            m1 = n1;
            l0 *= c0;
            l1 *= c1;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                O[k][0] *= c0;
                O[k][1] *= c1;
                O[k][2] *= c0;
                O[k][3] *= c1;
            }
            weigh();
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            l0 += w[k][0] + w[k][2];
            l1 += w[k][1] + w[k][3];
            if (!wide) kv4_tile_values<DT>(kaddr + KS_ROWS * KV4_ROW + k * 16 * KV4_ROW, sc[k], w[k], O);
            else kv4_tile_values_wide(kaddr + KS_ROWS * KV4_ROW + k * 16 * KV4_ROW, sc[k], w[k], O);
        }
        __syncwarp();   // (the stage is read: the next turn's copies go into it)
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    trace_last(p.ctl.trace, 2);
    __syncthreads();
    // ---- the warps' sums into one: under the largest reference
    float* sums = reinterpret_cast<float*>(smem);
    float* refs = sums + KS_WARPS * 8 * KS_SUM;   // [KS_WARPS][8] references, then as many sums of weights
    float* wsum = refs + KS_WARPS * 8;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, o);
        l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    if (2 * t < p.G) {
        float* row0 = sums + (warp * 8 + 2 * t) * KS_SUM;
        float* row1 = row0 + KS_SUM;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int d = kv4_dim_of(k, r);
            row0[d] = O[k][0];
            row1[d] = O[k][1];
            row0[d + 2] = O[k][2];
            row1[d + 2] = O[k][3];
        }
        if (r == 0) {
            refs[warp * 8 + 2 * t] = m0;
            refs[warp * 8 + 2 * t + 1] = m1;
            wsum[warp * 8 + 2 * t] = l0;
            wsum[warp * 8 + 2 * t + 1] = l1;
        }
    }
    if (CL) cluster_wait();
    __syncthreads();
    float* inbox = reinterpret_cast<float*>(smem + ks_inbox_at());
    const int own = (p.G + p.nsplit - 1) / p.nsplit;   // heads that a CTA finishes
    static_assert(KS_WARPS * 32 == HD, "a thread a dim");   // (heads and ranges unrolled: 4 x 9000 keys 9.0 us instead of 9.7)
    const int d = tid;
#pragma unroll 4
    for (int hh = 0; hh < p.G; hh++) {
        float M = KS_NONE;
#pragma unroll
        for (int w = 0; w < KS_WARPS; w++) M = fmaxf(M, refs[w * 8 + hh]);
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < KS_WARPS; w++) {
            const float f = ks_exp2(refs[w * 8 + hh] - M);
            num += sums[(w * 8 + hh) * KS_SUM + d] * f;
            den += wsum[w * 8 + hh] * f;
        }
        if (!CL) {
            // (no keys: zeros)
            Act<DT>::store(p.o, size_t(b) * p.o_stride + size_t(kvh * p.G + hh) * HD + d, den == 0.0f ? 0.0f : num / den);
        } else {
            const uint32_t row = cluster_map(smem_u32(inbox + (split * own + hh / p.nsplit) * KS_PART), uint32_t(hh % p.nsplit));
            cluster_st_f32(row + uint32_t(d) * 4u, num);
            if (d == 0) {
                cluster_st_f32(row + HD * 4, den);
                cluster_st_f32(row + (HD + 1) * 4, M);
            }
        }
    }
    if (CL) {
        // one cluster barrier: every range's rows are with their owners; CTA `split` finishes heads split, split + nsplit, ...
        cluster_arrive();
        cluster_wait();
        for (int slot = 0; slot < own; slot++) {
            const int hh = split + slot * p.nsplit;
            if (hh >= p.G) break;
            float M = KS_NONE, num = 0.0f, den = 0.0f;
            float refs_of[KS_MAX_CLUSTER];
#pragma unroll
            for (int k = 0; k < KS_MAX_CLUSTER; k++) {
                refs_of[k] = k < p.nsplit ? inbox[(k * own + slot) * KS_PART + HD + 1] : KS_NONE;
                M = fmaxf(M, refs_of[k]);
            }
#pragma unroll
            for (int k = 0; k < KS_MAX_CLUSTER; k++) {
                if (k >= p.nsplit) break;
                const float* row = inbox + (k * own + slot) * KS_PART;
                const float f = ks_exp2(refs_of[k] - M);
                num += row[d] * f;
                den += row[HD] * f;
            }
            Act<DT>::store(p.o, size_t(b) * p.o_stride + size_t(kvh * p.G + hh) * HD + d, den == 0.0f ? 0.0f : num / den);
        }
    }
    trace_last(p.ctl.trace, 3);
}

template <int DT, bool CL>
static EmblaStatus launch_kv4_sparse(EmblaAttn* ctx, const Kv4SparseParams& p, int batch, cudaStream_t s) {
    auto kern = kv4_sparse_kernel<DT, CL>;
    static bool configured[64] = {};   // per instantiation and device
    if (!configured[ctx->device & 63]) {
        // (the largest inbox: 7 ranges of 8 heads, two each)
        EMBLA_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(ks_smem(CL ? 7 : 1, 8))));
        configured[ctx->device & 63] = true;
    }
    const dim3 grid(p.nsplit, p.n_kv_heads, batch);
    EMBLA_CUDA_TRY(launch_kernel_cluster(ctx->pdl, CL ? p.nsplit : 1, kern, grid, dim3(KS_WARPS * 32), ks_smem(p.nsplit, p.G), s, p));
    EMBLA_CUDA_TRY(cudaGetLastError());
    return EMBLA_OK;
}

}  // namespace embla

using namespace embla;

extern "C" EmblaStatus embla_attn_sparse_decode_int4(EmblaAttn* ctx, const EmblaKVPool* pool, const EmblaKVView* view,
                                                     const EmblaQuery* q, const uint32_t* idx_dev, void* o_dev,
                                                     int64_t o_stride, void* stream) {
    if (!ctx || !pool || !view || !q || !q->q_dev || !o_dev) EMBLA_FAIL(EMBLA_BAD_ARG, "embla_attn_sparse_decode_int4: null argument");
    EMBLA_CHECK_DEVICE("embla_attn_sparse_decode_int4", ctx, pool);
    if (pool->kv_dtype != EMBLA_KV_INT4) EMBLA_FAIL(EMBLA_UNSUPPORTED, "embla_attn_sparse_decode_int4: the pool is not 4-bit");
    if (pool->n_kv_heads != ctx->cfg.n_kv_heads || view->layer < 0 || view->layer >= pool->n_layers)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_attn_sparse_decode_int4: pool/layer mismatch");
    if (view->batch <= 0 || view->batch > ctx->cfg.max_batch || !view->block_table_dev || !view->seq_lens_dev)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_attn_sparse_decode_int4: bad view (batch %d)", view->batch);
    if (!q->prenormed && (q->ng < 0 || q->ng > 2 || (q->ng >= 1 && !q->g1_dev) || (q->ng >= 2 && !q->g2_dev)))
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_attn_sparse_decode_int4: ng %d without its gain vectors", q->ng);
    const int max_len = view->max_seq_len > 0 ? view->max_seq_len : ctx->cfg.max_context;
    if (max_len > EMBLA_TOPK + EMBLA_RECENT && !idx_dev)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_attn_sparse_decode_int4: sequences past %d keys need the selected rows",
                   EMBLA_TOPK + EMBLA_RECENT);
    Kv4SparseParams p = {};
    p.pool = pool->base;
    p.block_table = view->block_table_dev;
    p.idx = idx_dev;
    p.seq_lens = view->seq_lens_dev;
    p.q = q->q_dev;
    p.g1 = q->g1_dev;
    p.g2 = q->g2_dev;
    p.o = o_dev;
    p.ctl = kernel_ctl(ctx);
    p.q_stride = q->q_stride;
    p.o_stride = o_stride;
    p.table_stride = view->table_stride;
    p.layer = view->layer;
    p.n_layers = pool->n_layers;
    p.n_kv_heads = pool->n_kv_heads;
    p.num_blocks = pool->num_blocks;
    p.G = ctx->cfg.n_q_heads / ctx->cfg.n_kv_heads;
    p.prenormed = q->prenormed;
    p.ng = q->ng;
    // CTAs a (sequence, kv head): what costs least in groups of rows a warp works through one after another, waves of CTAs
    // counted (four an SM), plus what a CTA costs beside them
    const int rows = max_len < EMBLA_TOPK + EMBLA_RECENT ? max_len : EMBLA_TOPK + EMBLA_RECENT;
    const long units = long(view->batch) * p.n_kv_heads, groups = (rows + KS_ROWS - 1) / KS_ROWS;
    long best = -1;
    for (int ns = 1; ns <= KS_MAX_CLUSTER && (ns == 1 || KS_WARPS * (ns - 1) < groups); ns++) {
        const long waves = (units * ns + 4 * ctx->sm_count - 1) / (4 * ctx->sm_count);
        const long cost = waves * ((groups + ns * KS_WARPS - 1) / (ns * KS_WARPS) + 4) + (ns > 1 ? 1 : 0);
        if (best < 0 || cost < best) {
            best = cost;
            p.nsplit = ns;
        }
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf = ctx->cfg.act_dtype == EMBLA_BF16;
    if (p.nsplit > 1) return bf ? launch_kv4_sparse<EMBLA_BF16, true>(ctx, p, view->batch, s) : launch_kv4_sparse<EMBLA_F16, true>(ctx, p, view->batch, s);
    return bf ? launch_kv4_sparse<EMBLA_BF16, false>(ctx, p, view->batch, s) : launch_kv4_sparse<EMBLA_F16, false>(ctx, p, view->batch, s);
}
