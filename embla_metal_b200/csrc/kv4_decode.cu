// Decode attention of the full layers over the 4-bit paged cache (EMBLA_KV_INT4): ReLU², one query token per sequence, with the
// key scores on request. No counterpart in the reference, whose cache is int8 (attn_full8, attention.metal:235-363).
//
// Bound by HBM: a key and its value are 144 bytes, used once. As in the int8 kernel (full_decode.cu) a CTA streams a range of a
// sequence's pages through a ring of shared-memory stages filled by TMA and a key's dots and sums run on warp tensor-core
// tiles (kv4_tile.cuh); per byte there are nearly twice as many codes to widen, so what counts is instructions a key:
// about 15 issue slots of the 25 that an SM has per key at full bandwidth.
//
// Weights. w = relu(q.k / sqrt(128))^2 has no bound, and its product with a value's scale goes through fp16. Each warp
// therefore keeps its weights as w' = relu(S)^2 f with a power of two f per head: when a weight of a tile passes LIMIT (tested
// with one vote a tile), f drops so that the tile's largest is TARGET or below, and the sums kept so far are scaled by the same power
// of two, exactly. Before the first key f is 2^100, so the first tile sets it. Weights between 2^10 and 2^13 at the top of
// their range leave 2^-24 / 2^10 of the largest as the smallest step; scales of 2 and more (values above 14) switch the
// warp to LIMIT 1/2, which no scale can push out of fp16.
#include <cstdlib>

#include "kv4_tile.cuh"

namespace embla {

constexpr int KD_PART = HD + 4;                                    // floats per (range, head): 128 sums, sum of weights
constexpr float KD_LIMIT = 8192.0f, KD_LIMIT_BIG = 0.5f;           // largest weight kept, usually and with large value scales
constexpr int KD_TARGET = 10, KD_TARGET_BIG = -4;                  // log2 of the bound a new f puts on the tile's weights
constexpr int KD_MAX_CLUSTER = 8;

struct Kv4DecodeParams {
    const uint8_t* pool;
    const int32_t* block_table;
    const int32_t* seq_lens;
    const void* q;
    const void* g1;
    const void* g2;
    void* o;
    float* partials;
    int* counters;
    KernelCtl ctl;
    float* scores;
    int64_t q_stride, o_stride, scores_stride;
    int table_stride, layer, n_layers, n_kv_heads, num_blocks, G, nsplit, prenormed, ng;
};

// shared memory: stages, queries, barriers, then (cluster launches) the rows [sender][head] that other ranges send
constexpr size_t kd_queries_at(int stages) { return size_t(stages) * KV4_PAGE; }
constexpr size_t kd_bars_at(int stages) { return kd_queries_at(stages) + sizeof(Kv4Queries); }
constexpr size_t kd_inbox_at(int stages) { return kd_bars_at(stages) + size_t(stages) * 20 + 12; }
constexpr size_t kd_inbox_rows(int ranges, int G) { return size_t(ranges) * ((G + ranges - 1) / ranges); }

// NCONS consumer warps share the 8 tiles of every page, the last warp is the producer. CL: the key ranges of a pair are the
// CTAs of one thread-block cluster, and each finishes the heads it owns (head h: CTA h % ranges) from its shared memory.
template <int DT, bool SCORES, int NCONS, int STAGES, int MINB, bool CL>
__global__ void __launch_bounds__((NCONS + 1) * 32, MINB)
    kv4_decode_kernel(const __grid_constant__ CUtensorMap tmap, const Kv4DecodeParams p) {
    constexpr int THREADS = (NCONS + 1) * 32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* stages = smem;
    Kv4Queries& sq = *reinterpret_cast<Kv4Queries*>(smem + kd_queries_at(STAGES));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kd_bars_at(STAGES));
    uint64_t* empty = full + STAGES;
    volatile int* limits = reinterpret_cast<volatile int*>(empty + STAGES);   // keys of the stage's page that count
    __shared__ int s_last, s_failed, s_issued;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    trace_first(p.ctl.trace, 0);
    if (CL) cluster_arrive();   // (every CTA of the cluster has started before any writes into another's shared memory)
    const int S = p.seq_lens[b];   // (an input of the whole step: read ahead of the wait)
    if (!p.ctl.early) {
        pdl_wait();
        pdl_launch_dependents();
    }
    const int npages = max(0, (S + BLK - 1) / BLK);
    const int pps = (npages + p.nsplit - 1) / p.nsplit;
    const int pg0 = split * pps;
    const int n = max(0, min(npages, pg0 + pps) - pg0);

    // ---- producer lane: page i of the range into its stage (a block outside the pool: no keys, and the error word set)
    auto issue = [&](int i, int block) {
        const int st = i % STAGES, use = i / STAGES;
        if (i == p.ctl.stall_at) return false;   // diagnostic stall: the consumers' wait for this page runs out
        if (use > 0 && !mbar_wait_bounded(p.ctl.wait_cycles, &empty[st], (use - 1) & 1)) {
            atomicExch(p.ctl.err, ERR_WAIT_EMPTY);
            return false;
        }
        if (block == -2) block = pg0 + i < p.table_stride ? p.block_table[size_t(b) * p.table_stride + pg0 + i] : -1;
        if (block < 0 || block >= p.num_blocks) {
            atomicExch(p.ctl.err, ERR_BAD_BLOCK);
            limits[st] = 0;
            mbar_arrive(&full[st]);
        } else {
            const long page = (long(block) * p.n_layers + p.layer) * p.n_kv_heads + kvh;
            uint8_t* dst = stages + st * KV4_PAGE;
            limits[st] = min(BLK, S - (pg0 + i) * BLK);
            mbar_expect_tx(&full[st], KV4_PAGE);
            tma_load_2d(dst, &tmap, 0, int(page * (KV4_PAGE / 128)), &full[st]);
            bulk_load_1d(dst + 2 * KV4_SIDE, p.pool + size_t(page) * KV4_PAGE + 2 * KV4_SIDE, KV4_SCALES, &full[st]);
        }
        *reinterpret_cast<volatile int*>(&s_issued) = i + 1;
        return true;
    };
    int next = 0;
    bool issuing = true;
    if (warp == NCONS) {
        const int ahead = min(n, STAGES);
        int myblock = -1;
        if (lane < ahead && pg0 + lane < p.table_stride) myblock = p.block_table[size_t(b) * p.table_stride + pg0 + lane];
        if (lane == 0) {
            for (int s = 0; s < STAGES; s++) {
                mbar_init(&full[s], 1);
                mbar_init(&empty[s], NCONS);
            }
            s_failed = 0;
            s_issued = 0;
            fence_barrier_init();
        }
        __syncwarp();
#pragma unroll
        for (int s = 0; s < STAGES; s++) {
            const int blk = __shfl_sync(0xffffffffu, myblock, s);
            if (lane == 0 && s < n && issuing) {
                issuing = issue(s, blk < 0 ? -1 : blk);
                next = s + 1;
            }
        }
    }
    if (p.ctl.early) {
        pdl_wait();
        pdl_launch_dependents();
    }
    trace_first(p.ctl.trace, 1);
    for (int hh = warp; hh < 8; hh += NCONS + 1)
        kv4_stage_query<DT>(sq, hh, hh < p.G, p.q, size_t(b) * p.q_stride + size_t(kvh * p.G + hh) * HD, p.prenormed != 0, p.g1, p.g2, p.ng, lane);
    __syncthreads();

    const int r = lane >> 2, t = lane & 3;
    float O[8][4];
#pragma unroll
    for (int i = 0; i < 8; i++) O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.0f;
    float ps0 = 0.0f, ps1 = 0.0f;                                   // sums of the kept weights of heads 2t, 2t + 1
    float f0 = pow2_biased(227), f1 = pow2_biased(227);             // their factors (2^100: nothing seen yet)

    if (warp == NCONS) {
        if (lane == 0)
            for (; next < n && issuing; next++) issuing = issue(next, -2);
    } else {
        Kv4Frag frag;
        frag.load(sq, lane);
        const uint32_t base = smem_u32(stages) + kv4_lane_at(lane);
        bool big = false;
        float limit = KD_LIMIT;
        // scores: S x the query's power of two; a head that is not there never is the largest
        float u0 = 0.0f, u1 = 0.0f, n0 = 0.0f, n1 = 0.0f;
        if (SCORES) {
            const int e0 = sq.expo[2 * t], e1 = sq.expo[2 * t + 1];
            if (e0) u0 = pow2_biased(e0);
            else n0 = __uint_as_float(0xff800000u);
            if (e1) u1 = pow2_biased(e1);
            else n1 = __uint_as_float(0xff800000u);
        }
        int st = 0, phase = 0;
        for (int i = 0; i < n; i++) {
            // (the decision is the warp's: a warp that leaves the loop leaves it whole)
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(p.ctl.wait_cycles, &full[st], phase))) {
                atomicExch(p.ctl.err, ERR_WAIT_FULL);
                *reinterpret_cast<volatile int*>(&s_failed) = 1;
                break;
            }
            const int lim = limits[st];
            const uint8_t* scales = stages + st * KV4_PAGE + 2 * KV4_SIDE;
#pragma unroll
            for (int step = 0; step < 8 / NCONS; step++) {
                const int R0 = (step * NCONS + warp) * 16;
                const int left = lim - R0;                          // keys of the tile that count, if under 16
                if (left <= 0) break;
                const uint32_t kaddr = base + st * KV4_PAGE + R0 * KV4_ROW;
                float s[4];
                kv4_tile_scores(kaddr, scales + R0 * 16, lane, frag, s);
                if (SCORES) {
                    float m0 = fmaxf(fmaf(s[0], u0, n0), fmaf(s[1], u1, n1)), m1 = fmaxf(fmaf(s[2], u0, n0), fmaf(s[3], u1, n1));
                    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 1));
                    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
                    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 2));
                    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 2));
                    const int key = r + 8 * t;
                    if (t < 2 && key < left)
                        p.scores[(size_t(b) * p.n_kv_heads + kvh) * p.scores_stride + (pg0 + i) * BLK + R0 + key] = t ? m1 : m0;
                }
                uint32_t vs[8];
                kv4_value_scales(scales + R0 * 16, lane, vs);
#pragma unroll
                for (int e = 0; e < 4; e++) s[e] = fmaxf(s[e], 0.0f);
                if (left < 16) {
                    if (r >= left) s[0] = s[1] = 0.0f;
                    if (r + 8 >= left) s[2] = s[3] = 0.0f;
                    kv4_mask_value_scales(vs, lane, left);
                }
                float w0 = s[0] * f0 * s[0], w1 = s[1] * f1 * s[1], w2 = s[2] * f0 * s[2], w3 = s[3] * f1 * s[3];
                const bool flagged = kv4_scales_large(vs);
                if (__any_sync(0xffffffffu, fmaxf(fmaxf(w0, w1), fmaxf(w2, w3)) > limit || (flagged && !big))) {
                    // (a handful of times a warp) new factors: the tile's largest weight of a head at most 2^target
                    if (__any_sync(0xffffffffu, flagged)) {
                        big = true;
                        limit = KD_LIMIT_BIG;
                    }
                    const int target = big ? KD_TARGET_BIG : KD_TARGET;
                    float m0 = fmaxf(s[0], s[2]), m1 = fmaxf(s[1], s[3]);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
                        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
                    }
                    // m < 2^(e + 1), so m^2 2^(target - 2 (e + 1)) < 2^target
                    const int e0 = int(__float_as_uint(m0) >> 23) - 126, e1 = int(__float_as_uint(m1) >> 23) - 126;
                    const float nf0 = m0 * f0 * m0 > limit ? pow2_biased(min(max(127 + target - 2 * e0, 1), 254)) : f0;
                    const float nf1 = m1 * f1 * m1 > limit ? pow2_biased(min(max(127 + target - 2 * e1, 1), 254)) : f1;
                    const float c0 = nf0 / f0, c1 = nf1 / f1;
                    f0 = nf0;
                    f1 = nf1;
                    ps0 *= c0;
                    ps1 *= c1;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        O[k][0] *= c0;
                        O[k][1] *= c1;
                        O[k][2] *= c0;
                        O[k][3] *= c1;
                    }
                    w0 = s[0] * f0 * s[0];
                    w1 = s[1] * f1 * s[1];
                    w2 = s[2] * f0 * s[2];
                    w3 = s[3] * f1 * s[3];
                }
                ps0 += w0 + w2;
                ps1 += w1 + w3;
                // the weights as fp16 (2^-11), keys across the lanes: the B registers of the sum
                kv4_tile_values(kaddr + KV4_SIDE, movmatrix4_trans(pack_h2(w0, w1)), movmatrix4_trans(pack_h2(w2, w3)), vs, O);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
            if (++st == STAGES) {
                st = 0;
                phase ^= 1;
            }
        }
    }

    trace_last(p.ctl.trace, 2);
    // ---- the warps' sums into one partial, in units of the weights themselves. The stages are free: every page that was
    // requested has been waited for, unless a wait gave up - then wait (bounded) for what is still in flight first.
    __syncthreads();
    if (s_failed) {
        if (tid == 0) {
            for (int i = max(0, s_issued - STAGES); i < s_issued; i++)
                if (!mbar_wait_bounded(p.ctl.wait_cycles, &full[i % STAGES], (i / STAGES) & 1)) atomicExch(p.ctl.err, ERR_WAIT_DRAIN);
        }
        __syncthreads();
    }
    float(*red)[8][HD] = reinterpret_cast<float(*)[8][HD]>(stages);
    float(*redp)[8] = reinterpret_cast<float(*)[8]>(stages + NCONS * 8 * HD * 4);
    if (warp < NCONS) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            ps0 += __shfl_xor_sync(0xffffffffu, ps0, o);
            ps1 += __shfl_xor_sync(0xffffffffu, ps1, o);
        }
        // w = w' / f x (the query's power of two)^2 / 128, the powers of two multiplied one by one
        const float q0 = pow2_biased(max(sq.expo[2 * t], 1)), q1 = pow2_biased(max(sq.expo[2 * t + 1], 1));
        const float i0 = (1.0f / 128.0f) / f0, i1 = (1.0f / 128.0f) / f1;
        auto real0 = [&](float x) { return x * i0 * q0 * q0; };
        auto real1 = [&](float x) { return x * i1 * q1 * q1; };
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int d = kv4_dim_of(k, r);
            red[warp][2 * t][d] = real0(O[k][0]);
            red[warp][2 * t + 1][d] = real1(O[k][1]);
            red[warp][2 * t][d + 2] = real0(O[k][2]);
            red[warp][2 * t + 1][d + 2] = real1(O[k][3]);
        }
        if (r == 0) {
            redp[warp][2 * t] = real0(ps0);
            redp[warp][2 * t + 1] = real1(ps1);
        }
    }
    __syncthreads();

    if (CL) cluster_wait();
    const int pair = b * p.n_kv_heads + kvh;
    const float sink = sqrtf(float(HD));
    float* part = p.partials + (size_t(pair) * p.nsplit + split) * p.G * KD_PART;
    float* inbox = reinterpret_cast<float*>(smem + kd_inbox_at(STAGES));
    const int slots = CL ? (p.G + p.nsplit - 1) / p.nsplit : 0;     // heads an owner finishes
    for (int idx = tid; idx < p.G * HD; idx += THREADS) {
        const int hh = idx >> 7, d = idx & 127;
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < NCONS; w++) {
            num += red[w][hh][d];
            den += redp[w][hh];
        }
        if (p.nsplit == 1) {
            Act<DT>::store(p.o, size_t(b) * p.o_stride + size_t(kvh * p.G + hh) * HD + d, num / (sink + den));
        } else if (CL) {
            const uint32_t row = cluster_map(smem_u32(inbox + (split * slots + hh / p.nsplit) * KD_PART), uint32_t(hh % p.nsplit));
            cluster_st_f32(row + uint32_t(d) * 4u, num);
            if (d == 0) cluster_st_f32(row + HD * 4, den);
        } else {
            part[hh * KD_PART + d] = num;
            if (d == 0) part[hh * KD_PART + HD] = den;
        }
    }
    if (p.nsplit == 1) {
        trace_last(p.ctl.trace, 3);
        return;
    }
    if (CL) {
        cluster_arrive();
        cluster_wait();
        for (int idx = tid; idx < slots * HD; idx += THREADS) {
            const int slot = idx >> 7, d = idx & 127, hh = split + slot * p.nsplit;
            if (hh < p.G) {
                float num = 0.0f, den = sink;
                for (int k = 0; k < p.nsplit; k++) {
                    const float* row = inbox + (k * slots + slot) * KD_PART;
                    den += row[HD];
                    num += row[d];
                }
                Act<DT>::store(p.o, size_t(b) * p.o_stride + size_t(kvh * p.G + hh) * HD + d, num / den);
            }
        }
        trace_last(p.ctl.trace, 3);
        return;
    }
    // last CTA of the pair to arrive adds the ranges in order (arrive_last, common.metal:88-99)
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        const int prev = atomicAdd(&p.counters[pair], 1);
        s_last = prev == p.nsplit - 1;
        if (s_last) p.counters[pair] = 0;
    }
    __syncthreads();
    if (!s_last) {
        trace_last(p.ctl.trace, 3);
        return;
    }
    __threadfence();
    const float* all = p.partials + size_t(pair) * p.nsplit * p.G * KD_PART;
    const int n4 = p.nsplit * p.G * (KD_PART / 4);
    const bool staged = n4 * 16 <= STAGES * KV4_PAGE;
    if (staged) {
        stage_from_global<THREADS>(reinterpret_cast<float4*>(stages), reinterpret_cast<const float4*>(all), n4, tid);
        __syncthreads();
        all = reinterpret_cast<const float*>(stages);
    }
    for (int idx = tid; idx < p.G * HD; idx += THREADS) {
        const int hh = idx >> 7, d = idx & 127;
        float num = 0.0f, den = sink;
        for (int k = 0; k < p.nsplit; k++) {
            const float* row = all + (size_t(k) * p.G + hh) * KD_PART;
            den += staged ? row[HD] : __ldcg(row + HD);
            num += staged ? row[d] : __ldcg(row + d);
        }
        Act<DT>::store(p.o, size_t(b) * p.o_stride + size_t(kvh * p.G + hh) * HD + d, num / den);
    }
    trace_last(p.ctl.trace, 3);
}

int choose_full_decode_split(int pairs, int pages, int slots, int max_slots, bool* cluster);   // full_decode.cu

constexpr int KD_NCONS = 4, KD_STAGES = 3, KD_MINB = 3;

template <int DT, bool SCORES, bool CL>
static EmblaStatus launch_kv4_decode(EmblaAttn* ctx, const EmblaKVPool* pool, const Kv4DecodeParams& p, int batch, cudaStream_t s) {
    auto kern = kv4_decode_kernel<DT, SCORES, KD_NCONS, KD_STAGES, KD_MINB, CL>;
    const size_t smem = 1024 + kd_inbox_at(KD_STAGES) + (CL ? kd_inbox_rows(p.nsplit, p.G) * KD_PART * 4 : 0);
    static bool configured[64] = {};   // per instantiation and device
    if (!configured[ctx->device & 63]) {
        // (the largest inbox: 7 ranges of 8 heads, two each)
        EMBLA_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            int(1024 + kd_inbox_at(KD_STAGES) + (CL ? 14 * KD_PART * 4 : 0))));
        configured[ctx->device & 63] = true;
    }
    const dim3 grid(p.nsplit, p.n_kv_heads, batch);
    EMBLA_CUDA_TRY(launch_kernel_cluster(ctx->pdl, CL ? p.nsplit : 1, kern, grid, dim3((KD_NCONS + 1) * 32), smem, s, pool->tmap_codes, p));
    EMBLA_CUDA_TRY(cudaGetLastError());
    return EMBLA_OK;
}

EmblaStatus kv4_full_decode(EmblaAttn* ctx, const EmblaKVPool* pool, const EmblaKVView* view, const EmblaQuery* q, void* o_dev,
                            int64_t o_stride, float* scores_dev, int64_t scores_stride, int max_len, cudaStream_t stream) {
    Kv4DecodeParams p = {};
    p.pool = pool->base;
    p.block_table = view->block_table_dev;
    p.seq_lens = view->seq_lens_dev;
    p.q = q->q_dev;
    p.g1 = q->g1_dev;
    p.g2 = q->g2_dev;
    p.o = o_dev;
    p.partials = ctx->partials;
    p.counters = ctx->counters;
    p.ctl = kernel_ctl(ctx);
    p.scores = scores_dev;
    p.q_stride = q->q_stride;
    p.o_stride = o_stride;
    p.scores_stride = scores_stride;
    p.table_stride = view->table_stride;
    p.layer = view->layer;
    p.n_layers = pool->n_layers;
    p.n_kv_heads = pool->n_kv_heads;
    p.num_blocks = pool->num_blocks;
    p.G = ctx->cfg.n_q_heads / ctx->cfg.n_kv_heads;
    p.prenormed = q->prenormed;
    p.ng = q->ng;
    const int pairs = view->batch * pool->n_kv_heads, pages = (max_len + BLK - 1) / BLK;
    bool cluster = false;
    p.nsplit = choose_full_decode_split(pairs, pages, KD_MINB * ctx->sm_count, ctx->partial_slots, &cluster);
    const bool bf = ctx->cfg.act_dtype == EMBLA_BF16;
#define EMBLA_KD(DT, SC) (cluster ? launch_kv4_decode<DT, SC, true>(ctx, pool, p, view->batch, stream) \
                                  : launch_kv4_decode<DT, SC, false>(ctx, pool, p, view->batch, stream))
    if (scores_dev) return bf ? EMBLA_KD(EMBLA_BF16, true) : EMBLA_KD(EMBLA_F16, true);
    return bf ? EMBLA_KD(EMBLA_BF16, false) : EMBLA_KD(EMBLA_F16, false);
#undef EMBLA_KD
}

}  // namespace embla
