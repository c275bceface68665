// Decode attention of the full layers over the 4-bit paged cache (EMBLA_KV_INT4): ReLU², one query token per sequence, with the
// key scores on request. No counterpart in the reference, whose cache is int8 (attn_full8, attention.metal:235-363).
//
// Bound by HBM: a key and its value are 144 bytes, used once. As in the int8 kernel (full_decode.cu) a CTA streams a range of a
// sequence's pages through a ring of shared-memory stages filled by TMA and a key's dots and sums run on warp tensor-core
// tiles (kv4_tile.cuh); per byte there are nearly twice as many codes to widen, so what counts is instructions a key:
// about 17.9 for fp16 outputs, 16.5 for bf16, of the 25 issue slots that an SM has per key at full bandwidth, 7.5 of them on the ALU
// pipe, which has 12. 64 sequences of 32768 keys, 4 kv heads: 224 to 260 us (fp16, 4.6 to 5.4 TB/s, 0.71 to 0.82 of the measured copy rate;
// it differs from GPU to GPU and with the values that the cache holds) and 9 to 12 us less in bf16; 16 uneven sequences of up to 9001 keys: 26 to 28 us;
// one of 1000: 6.6 us. What is left of it: half of the issue slots
// are used, twelve warps being what 128 registers a thread leave room for; a launch's first 4 microseconds (lengths, block
// table, first pages one after another) and its last 3 (the pieces' sums, written on one SM and read on another). Adding the
// pieces up in the CTA that ends last, counted by atomics, took 0.7 to 2 microseconds longer than a second launch that is there
// and waits; running the page loop once ahead of the first page, for the instruction caches, 1.3 longer than not.
//
// Weights. w = relu(q.k / sqrt(128))^2 has no bound, and its product with a value's scale goes through fp16. Each warp
// therefore keeps its weights as w' = relu(S)^2 f with a power of two f per head: when a weight of a tile passes LIMIT (tested
// with one vote a tile), f drops so that the tile's largest is TARGET or below, and the sums kept so far are scaled by the same power
// of two, exactly. Before the first key f is 2^120, so the first tile sets it. Weights between 2^10 and 2^13 at the top of
// their range leave 2^-24 / 2^10 of the largest as the smallest step. A tile with a value scale of 8 or more (values above 56), whose
// product with a weight fp16 may not hold, takes its products in two bf16 parts (kv4_tile_values_wide).
#include <cstdlib>

#include "kv4_tile.cuh"

namespace embla {

// The same value, computed here: what hangs on it is not worked out ahead of the loop around it and kept in registers meanwhile.
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+r"(x));
    return x;
}
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

__device__ __forceinline__ void prefetch_tensormap(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void* at) { asm volatile("prefetch.global.L2 [%0];" ::"l"(at)); }

// a barrier that tells all its threads whether any of them said yes
__device__ __forceinline__ bool bar_any(int id, int threads, bool yes) {
    int any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.s32 p, %1, 0;\n bar.red.or.pred q, %2, %3, p;\n selp.s32 %0, 1, 0, q;\n}\n"
        : "=r"(any)
        : "r"(int(yes)), "r"(id), "r"(threads)
        : "memory");
    return any != 0;
}

constexpr int KD_PART = HD + 4;                                    // floats per (range, head): 128 sums, sum of weights
constexpr int KD_SUM = HD + 1;   // a row of a warp's sums in shared memory: lanes (r, t) write heads 2t at dims 8 (r / 2) + r % 2: 32 banks
constexpr float KD_LIMIT = 8192.0f;                                // largest weight kept
constexpr int KD_TARGET = 10;                                      // log2 of the bound a new f puts on the tile's weights
constexpr int KD_MAX_CLUSTER = 8;
// What a unit costs beside its pages, in pages (16 uneven sequences of up to 9001 keys, where 4 take 26 to 28 us: 2.7 us more counting 2, 10 more
// counting none).
constexpr int KD_UNIT_COST = 4;
constexpr int KD_MIN_RUN = 4;   // cost of a run at least

struct Kv4DecodeParams {
    const uint8_t* pool;
    const int32_t* block_table;
    const int32_t* seq_lens;
    const void* q;
    const void* g1;
    const void* g2;
    void* o;
    float* partials;
    KernelCtl ctl;
    float* scores;
    int64_t q_stride, o_stride, scores_stride;
    int table_stride, layer, n_layers, n_kv_heads, num_blocks, G, batch, nsplit, n_runs, prenormed, ng;
};

constexpr int KD_HELPERS = 3;
struct KdSlot;
constexpr int kd_bufs(bool cl) { return cl ? 1 : 4; }   // pieces staged ahead
// shared memory: stages, slots, barriers, the warps' sums, then (cluster launches) the rows [sender][head] of the other ranges
constexpr size_t KD_SLOT_BYTES = sizeof(Kv4Queries) + 16;
constexpr size_t kd_slots_at(int stages) { return size_t(stages) * KV4_PAGE; }
constexpr size_t kd_bars_at(int stages, bool cl) { return kd_slots_at(stages) + kd_bufs(cl) * KD_SLOT_BYTES; }
constexpr size_t kd_sums_at(int stages, bool cl) { return (kd_bars_at(stages, cl) + size_t(stages) * 20 + (2 * kd_bufs(cl) + 4) * 8 + 15) / 16 * 16; }
constexpr size_t kd_smem(int ncons, int stages, bool cl) { return 1024 + kd_sums_at(stages, cl) + size_t(ncons) * 8 * KD_SUM * 4; }
constexpr size_t kd_inbox_rows(int ranges, int G) { return size_t(ranges) * ((G + ranges - 1) / ranges); }

__device__ __forceinline__ int kd_pages(const int32_t* seq_lens, int b) {
    const int S = __ldg(seq_lens + b);
    return S > 0 ? (S - 1) / BLK + 1 : 0;
}

// What a unit of that many pages counts for when the work is cut: a unit begins with KD_UNIT_COST counts that stand for no page.
__device__ __forceinline__ unsigned kd_cost(int pages) { return pages > 0 ? unsigned(pages + KD_UNIT_COST) : 0u; }

// The costs of all units, laid end to end, cut into `runs` runs whose lengths differ by one at most (and are KD_MIN_RUN or more,
// so that fewer CTAs than launched may have one).
struct KdRuns {
    unsigned runs, len, longer;   // the first `longer` runs are len + 1 long, the others len
    __device__ __forceinline__ KdRuns(unsigned cost, unsigned most) {
        runs = max(1u, min(most, (cost + KD_MIN_RUN - 1) / KD_MIN_RUN));
        len = cost / runs;
        longer = cost - len * runs;
    }
    __device__ __forceinline__ unsigned start_of(unsigned c) const { return c * len + min(c, longer); }
    __device__ __forceinline__ unsigned run_of(unsigned x) const {   // the run that count x is in
        const unsigned edge = longer * (len + 1);
        return x < edge ? x / (len + 1) : longer + (x - edge) / max(len, 1u);
    }
};

// A piece of work: pages [first, first + n) of a unit (sequence b, kv head kvh) that has `pages` of them.
struct KdPiece {
    int b, kvh, first, n, pages;
};

// The work of a CTA, walked by its producer and its helpers alike. CL: the one range that the launch grid gives it. Else the costs
// of all units, laid end to end (by sequence, then kv head), are cut into equal runs, one a CTA, whatever the sequences'
// lengths: a run may end and begin inside a unit, whose pieces then meet in the scratch.
template <bool CL>
struct KdWalk {
    int left;        // cost of the run still to come
    int into;        // where in the unit `at` stands at its next piece begins, in cost
    int pieces;      // of the run so far
    KdPiece at;      // piece under way

    __device__ __forceinline__ void start(const Kv4DecodeParams& p, int lane) {
        left = into = pieces = 0;
        at.n = 0;
        if (CL) {
            at.b = blockIdx.z;
            at.kvh = blockIdx.y;
            at.pages = kd_pages(p.seq_lens, at.b);
            const int per = (at.pages + p.nsplit - 1) / p.nsplit;
            at.first = int(blockIdx.x) * per;
            left = max(0, min(at.pages, at.first + per) - at.first);
            return;
        }
        // (up to 32 sequences, the usual case, take one load of their lengths)
        auto scan = [&](int i0, unsigned& n, int& pages) {
            pages = i0 + lane < p.batch ? kd_pages(p.seq_lens, i0 + lane) : 0;
            n = kd_cost(pages);
            unsigned incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            return incl;
        };
        unsigned n, incl;
        int pages;
        incl = scan(0, n, pages);
        unsigned sum = __shfl_sync(0xffffffffu, incl, 31);
        for (int i = 32 + lane; i < (p.batch + 31) / 32 * 32; i += 32)
            sum += __reduce_add_sync(0xffffffffu, i < p.batch ? kd_cost(kd_pages(p.seq_lens, i)) : 0u);
        const KdRuns cut(sum * p.n_kv_heads, p.n_runs);
        const unsigned c = blockIdx.x;
        if (c >= cut.runs) return;
        const unsigned x0 = cut.start_of(c);
        left = int(cut.start_of(c + 1) - x0);
        // the sequence that count x0 falls in: the first one whose units end behind it
        unsigned before = 0;
        for (int i0 = 0; i0 < p.batch; i0 += 32) {
            if (i0 > 0) incl = scan(i0, n, pages);
            const unsigned here = __ballot_sync(0xffffffffu, (before + incl) * p.n_kv_heads > x0);
            if (here) {
                const int l = __ffs(here) - 1;
                const unsigned cost = __shfl_sync(0xffffffffu, n, l);
                at.b = i0 + l;
                at.pages = __shfl_sync(0xffffffffu, pages, l);
                const unsigned in = x0 - (before + __shfl_sync(0xffffffffu, incl, l) - cost) * p.n_kv_heads;
                at.kvh = int(in / cost);
                into = int(in - unsigned(at.kvh) * cost);
                return;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    // the next piece of the run; false when it is done
    __device__ __forceinline__ bool next(const Kv4DecodeParams& p) {
        if (CL) {
            if (left <= 0) return false;
            at.n = left;
            left = 0;
            return true;
        }
        while (left > 0) {
            if (into == at.pages + KD_UNIT_COST) {   // behind the last unit
                into = 0;
                if (++at.kvh == p.n_kv_heads) {
                    at.kvh = 0;
                    do at.pages = kd_pages(p.seq_lens, ++at.b);
                    while (at.pages == 0);   // (the run is not done: a sequence that has pages follows)
                }
            }
            const int take = min(left, at.pages + KD_UNIT_COST - into);
            at.first = max(0, into - KD_UNIT_COST);
            at.n = max(0, into + take - KD_UNIT_COST) - at.first;
            into += take;
            left -= take;
            if (at.n > 0) {
                pieces++;
                return true;
            }
        }
        at.n = 0;
        return false;
    }
};

// A piece as the helper warps hand it to the consumers: its queries, and what of it is to be done.
struct KdSlot {
    Kv4Queries sq;
    int n;         // pages; -1: there are no more pieces
    int first;     // its first page in the sequence
    int unit;      // sequence x kv heads + kv head
    int out;       // -1: the unit is whole in this run; else the slot of the scratch that its sums go to
};

// NCONS consumer warps; a producer warp; HELPERS helper warps. WPG consumer warps share the 8 tiles of a page; the NCONS / WPG
// groups of them take the run's pages in turn, so that no group gets far ahead of another (three CTAs an SM with a run each did:
// the warps of the one that the schedulers favoured were done after 0.8 of the time, and the others were left with too few warps
// for the SM). The helpers stage the queries of the next pieces and write out the sums of the last ones, so that a piece costs
// the consumers a look at its slot, and short pieces (a page or two) are worked on by several groups at a time; with the consumers
// doing that work between barriers a piece cost 3.7 microseconds beside its pages.
// CL: the key ranges of a unit are the CTAs of one thread-block cluster, and each finishes the heads it owns (head h: CTA h %
// ranges) from its shared memory.
static_assert(sizeof(KdSlot) == KD_SLOT_BYTES && KD_SLOT_BYTES % 16 == 0, "the slots' place in shared memory");

template <int DT, bool SCORES, int NCONS, int WPG, int STAGES, bool CL>
__global__ void __launch_bounds__((NCONS + 1 + KD_HELPERS) * 32, 1)
    kv4_decode_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ Kv4DecodeParams p) {
    constexpr int TILES = 8 / WPG;          // 16-key tiles of a page a consumer warp takes
    // of those, taken together: all (one by one 64 x 32768 keys take 7 % longer), but one by one where scores are written
    // too, which leaves no registers for two (8 x 32768 keys, where one by one takes 28.8 to 30.8 us: 1 us more)
    constexpr int STEP = SCORES ? 1 : TILES;
    constexpr int GROUPS = NCONS / WPG;
    constexpr int PRODUCER = NCONS;         // warp roles: consumers, then the producer, then the helpers
    constexpr int BUFS = kd_bufs(CL);
    // Pages in flight until the first ones are there: the whole ring requested at once by all CTAs is 4 microseconds of the HBM's
    // time, and the first pages of a CTA come as late as the last (64 sequences of 1000 keys: 20.1 us with three in flight, 21.3
    // with five, 22.7 with nine; a lone cluster's CTA has few and takes all it can).
    constexpr int AHEAD = CL ? STAGES : GROUPS;
    static_assert(STAGES >= GROUPS, "a group's stage index advances by GROUPS a page");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* stages = smem;
    KdSlot* slots = reinterpret_cast<KdSlot*>(smem + kd_slots_at(STAGES));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kd_bars_at(STAGES, CL));
    uint64_t* empty = full + STAGES;
    uint64_t* staged = empty + STAGES;      // [BUFS] helpers -> consumers: the slot holds a piece
    uint64_t* summed = staged + BUFS;       // [BUFS] consumers -> helpers: all are past the slot's piece, its sums written
    uint64_t* taken = summed + BUFS;        // [GROUPS] helpers -> the group: its sums have been read
    volatile int* limits = reinterpret_cast<volatile int*>(taken + GROUPS);   // [STAGES] keys of the stage's page that count
    float* sums = reinterpret_cast<float*>(smem + kd_sums_at(STAGES, CL));    // [NCONS][8][KD_SUM]
    __shared__ int s_failed, s_issued;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    trace_first(p.ctl.trace, 0);
    if (CL) cluster_arrive();   // (every CTA of the cluster has started before any writes into another's shared memory)
    auto fail = [&](int code) {
        atomicExch(p.ctl.err, code);
        *reinterpret_cast<volatile int*>(&s_failed) = 1;
    };

    if (warp == PRODUCER) {
        // ---- producer: keeps the ring of stages full. The lanes look up 32 pages' blocks and addresses at a time, then each requests
        // its page when its turn comes (one lane that did it all took 1000 clocks a page, twice what the SM takes to attend one).
        // A block outside the pool: no keys, and the error word set.
        KdWalk<CL> walk;
        if (lane == 0) prefetch_tensormap(&tmap);
        walk.start(p, lane);                // (reads the sequence lengths ahead of the wait: nothing on the GPU writes them)
        if (lane == 0) {
            for (int s = 0; s < STAGES; s++) {
                mbar_init(&full[s], 1);
                mbar_init(&empty[s], WPG);
            }
            for (int s = 0; s < BUFS; s++) {
                mbar_init(&staged[s], KD_HELPERS);
                mbar_init(&summed[s], NCONS);
            }
            for (int s = 0; s < GROUPS; s++) mbar_init(&taken[s], KD_HELPERS);
            s_failed = 0;
            fence_barrier_init();
        }
        pdl_wait();
        pdl_launch_dependents();
        int count = 0, done = 0, S = 0;     // pages requested, of the run and of the piece; keys of the sequence
        bool go = true, joined = false;
        while (true) {
            if (go && done == walk.at.n) {
                go = walk.next(p);
                done = 0;
                S = go ? __ldg(p.seq_lens + walk.at.b) : 0;
            }
            if (!joined && (!go || count >= AHEAD)) {   // (none of it waited for a barrier so far)
                __syncthreads();
                joined = true;
            }
            if (!go) break;
            const int m = min(min(32, walk.at.n - done), joined ? 32 : AHEAD - count);
            const int page = walk.at.first + done + lane, mine = count + lane, st = mine % STAGES;
            const int block = lane < m && page < p.table_stride ? p.block_table[size_t(walk.at.b) * p.table_stride + page] : -1;
            const bool there = block >= 0 && block < p.num_blocks;
            const long pg = (long(block) * p.n_layers + p.layer) * p.n_kv_heads + walk.at.kvh;
            const uint8_t* scales = p.pool + size_t(pg) * KV4_PAGE + 2 * KV4_SIDE;
            uint8_t* dst = stages + st * KV4_PAGE;
            for (int i = 0; i < m && go; i++) {
                bool bad = false;
                if (lane == i) {
                    if (mine == p.ctl.stall_at) {   // diagnostic stall: the consumers' wait for this page runs out
                        bad = true;
                    } else if (mine >= STAGES && !mbar_wait_bounded(p.ctl.wait_cycles, &empty[st], (mine / STAGES - 1) & 1)) {
                        atomicExch(p.ctl.err, ERR_WAIT_EMPTY);
                        bad = true;
                    } else if (mine >= AHEAD && mine < STAGES && !mbar_wait_bounded(p.ctl.wait_cycles, &full[mine - AHEAD], 0)) {
                        atomicExch(p.ctl.err, ERR_WAIT_FULL);
                        bad = true;
                    } else if (there) {
                        limits[st] = min(BLK, S - page * BLK);
                        mbar_expect_tx(&full[st], KV4_PAGE);
                        tma_load_2d(dst, &tmap, 0, int(pg * (KV4_PAGE / 128)), &full[st]);
                        bulk_load_1d(dst + 2 * KV4_SIDE, scales, KV4_SCALES, &full[st]);
                    } else {
                        atomicExch(p.ctl.err, ERR_BAD_BLOCK);
                        limits[st] = 0;
                        if (SCORES) {   // (its scores are zeros, not an earlier call's)
                            float* row = p.scores + size_t(walk.at.b * p.n_kv_heads + walk.at.kvh) * p.scores_stride + long(page) * BLK;
                            for (int key = min(BLK, S - page * BLK) - 1; key >= 0; key--) row[key] = 0.0f;
                        }
                        mbar_arrive(&full[st]);
                    }
                }
                go = !__any_sync(0xffffffffu, bad);
                count += go ? 1 : 0;
            }
            done += m;
        }
        if (lane == 0) s_issued = count;
    } else if (warp > PRODUCER) {
        // ---- helpers: warp hw stages heads hw, hw + KD_HELPERS, ..; the sums are shared out by thread
        const int hw = warp - PRODUCER - 1, ht = hw * 32 + lane;
        constexpr int HPW = (8 + KD_HELPERS - 1) / KD_HELPERS;      // heads a helper warp takes
        KdWalk<CL> walk;
        walk.start(p, lane);
        bool more = true;
        pdl_wait();
        float x[HPW][4];                    // the warp's query rows of the next piece, on their way since the one before it was staged
        auto fetch = [&]() {
            more = walk.next(p) || (CL && more);   // (a range without pages sends its zeros all the same)
            const size_t row = size_t(walk.at.b) * p.q_stride + size_t(walk.at.kvh * p.G) * HD;
#pragma unroll
            for (int i = 0; i < HPW; i++) kv4_load_query<DT>(x[i], more && hw + i * KD_HELPERS < p.G, p.q, row + size_t(hw + i * KD_HELPERS) * HD, lane);
        };
        auto stage = [&](int j) {
            KdSlot& slot = slots[j % BUFS];
#pragma unroll
            for (int i = 0; i < HPW; i++) {
                const int hh = hw + i * KD_HELPERS;
                if (hh < 8) kv4_stage_query<DT>(slot.sq, hh, hh < p.G, x[i], p.prenormed != 0, p.g1, p.g2, p.ng, lane);
            }
            if (ht == 0) {
                const KdPiece& at = walk.at;
                slot.n = more ? at.n : -1;
                slot.first = at.first;
                slot.unit = at.b * p.n_kv_heads + at.kvh;
                // a run has at most two pieces of units that it shares with others, its first and its last
                slot.out = at.n == at.pages ? -1 : 2 * int(blockIdx.x) + (walk.pieces == 1 ? 0 : 1);
            }
        };
        fetch();
        int ahead = 0;
        stage(ahead++);
        __syncthreads();
        if (lane == 0) mbar_arrive(&staged[0]);
        if (!CL) {
            bool last = !more;              // the slot without pages has been staged
            if (!last) fetch();
            for (int c = blockIdx.x; c < p.batch; c += gridDim.x)   // sequences without keys have no unit in any run
                if (__ldg(p.seq_lens + c) <= 0)
                    for (int i = ht; i < p.n_kv_heads * p.G * HD; i += KD_HELPERS * 32) Act<DT>::store(p.o, size_t(c) * p.o_stride + i, 0.0f);
            const float sink = sqrtf(float(HD));
            int piece0 = 0;
#pragma unroll 1
            for (int j = 0;; j++) {
                // up to BUFS pieces ahead of the one whose sums come next
                for (; !last && ahead < j + BUFS; ahead++) {
                    stage(ahead);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&staged[ahead % BUFS]);
                    last = !more;
                    if (!last) fetch();
                }
                const KdSlot& slot = slots[j % BUFS];
                bar_sync(2, KD_HELPERS * 32);                       // (the slot's words are thread 0's)
                const int n = slot.n;
                if (n < 0) break;
                // (the helpers go on or leave together: the barriers below count all of them)
                if (bar_any(2, KD_HELPERS * 32, !mbar_wait_bounded(p.ctl.wait_cycles, &summed[j % BUFS], (j / BUFS) & 1))) {
                    fail(ERR_WAIT_FULL);
                    break;
                }
                const int out = slot.out, unit = slot.unit;
                // the groups that had a page of the piece: those of pages piece0 .. piece0 + n - 1
                const int g0 = piece0 % GROUPS;
                auto has = [&](int g) { return (g - g0 + GROUPS) % GROUPS < n; };
                for (int hh = hw; hh < p.G; hh += KD_HELPERS) {
                    float num[4] = {0.0f, 0.0f, 0.0f, 0.0f}, den = 0.0f;   // dims lane + 32 i
#pragma unroll
                    for (int g = 0; g < GROUPS; g++) {
                        if (!has(g)) continue;
#pragma unroll
                        for (int w = 0; w < WPG; w++) {
                            const float* from = sums + ((g * WPG + w) * 8 + hh) * KD_SUM;
#pragma unroll
                            for (int i = 0; i < 4; i++) num[i] += from[lane + 32 * i];
                            den += from[HD];
                        }
                    }
                    if (out < 0) {
                        const size_t at = size_t(unit / p.n_kv_heads) * p.o_stride + size_t(unit % p.n_kv_heads * p.G + hh) * HD + lane;
#pragma unroll
                        for (int i = 0; i < 4; i++) Act<DT>::store(p.o, at + 32 * i, num[i] / (sink + den));
                    } else {
                        float* part = p.partials + (size_t(out) * p.G + hh) * KD_PART;
#pragma unroll
                        for (int i = 0; i < 4; i++) part[lane + 32 * i] = num[i];
                        if (lane == 0) part[HD] = den;
                    }
                }
                __syncwarp();
                if (lane == 0)
                    for (int g = 0; g < GROUPS; g++)
                        if (has(g)) mbar_arrive(&taken[g]);
                piece0 += n;
                bar_sync(2, KD_HELPERS * 32);                       // (all are done with the slot: it may be staged again)
            }
        }
    } else {
        // ---- consumers
        if (!CL) {
            // the block tables on their way to the L2 while the producers look for their runs (16 uneven sequences of up to 9001 keys, 26 to 28 us:
            // 0.4 us less)
            const long at = (long(blockIdx.x) * NCONS + warp) * 1024 + lane * 32;   // a line of 32 entries a lane
            if (at <= long(p.batch - 1) * p.table_stride) prefetch_l2(p.block_table + at);
        }
        pdl_wait();
        trace_first(p.ctl.trace, 1);
        const int r = lane >> 2, t = lane & 3;
        const uint32_t base = smem_u32(stages) + kv4_lane_at(lane);
        const int group = warp / WPG, wg = warp % WPG;
        int st = group, phase = 0;                                  // stage and phase of the group's next page,
        int mine = group, piece0 = 0;                               // its number in the run, and of the piece's first page
        int given = 0;                                              // pieces that the group has left sums of
        __syncthreads();
#pragma unroll 1
        for (int j = 0;; j++) {
            const KdSlot& slot = slots[j % BUFS];
            // (the decision is the warp's, here and below: a warp that leaves a loop leaves it whole)
            bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(p.ctl.wait_cycles, &staged[j % BUFS], (j / BUFS) & 1));
            if (!ok) {
                fail(ERR_WAIT_FULL);
                break;
            }
            const int n = slot.n;
            if (n < 0) break;
            if (CL || mine < piece0 + n) {
                Kv4Frag frag;
                frag.load(slot.sq, here(lane));
                // scores: S x the query's power of two; a head that is not there never is the largest
                float u0 = 0.0f, u1 = 0.0f, n0 = 0.0f, n1 = 0.0f;
                float* scores = nullptr;
                if (SCORES) {
                    const int e0 = slot.sq.expo[2 * t], e1 = slot.sq.expo[2 * t + 1];
                    if (e0) u0 = pow2_biased(e0) / KV4_SUBNORMAL;
                    else n0 = __uint_as_float(0xff800000u);
                    if (e1) u1 = pow2_biased(e1) / KV4_SUBNORMAL;
                    else n1 = __uint_as_float(0xff800000u);
                    scores = p.scores + size_t(slot.unit) * p.scores_stride + long(slot.first - piece0) * BLK + wg * (TILES * 16);
                }
                float O[8][4];
#pragma unroll
                for (int i = 0; i < 8; i++) O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.0f;
                float ps0 = 0.0f, ps1 = 0.0f;                       // sums of the kept weights of heads 2t, 2t + 1
                float f0 = pow2_biased(247), f1 = pow2_biased(247); // their factors (2^120: nothing seen yet)
#pragma unroll 1
                for (; mine < piece0 + n; mine += GROUPS) {
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(p.ctl.wait_cycles, &full[st], phase));
                    if (!ok) break;
                    // the tiles of a step together: their products have nothing to wait for in one another
                    const uint32_t kaddr0 = base + st * KV4_PAGE + wg * (TILES * 16 * KV4_ROW);
                    const uint8_t* sc0 = stages + st * KV4_PAGE + 2 * KV4_SIDE + wg * (TILES * 16 * 16);
                    const int left0 = limits[st] - wg * (TILES * 16);   // keys of the tiles that count, if fewer than there are
#pragma unroll
                    for (int tile = 0; tile < TILES; tile += STEP) {
                        const uint32_t kaddr = kaddr0 + tile * 16 * KV4_ROW;
                        const uint8_t* sc = sc0 + tile * 256;
                        const int left = left0 - tile * 16;
                        if (left > 0) {
                            float s[STEP][4];
                            Kv4Scales rows[STEP];
                            bool flagged = false;
#pragma unroll
                            for (int k = 0; k < STEP; k++) {
                                rows[k].load(sc + k * 256, lane);
                                kv4_tile_scores(kaddr + k * 16 * KV4_ROW, rows[k], frag, s[k]);
                            }
                            if (SCORES) {
#pragma unroll
                                for (int k = 0; k < STEP; k++) {
                                    float m0 = fmaxf(fmaf(s[k][0], u0, n0), fmaf(s[k][1], u1, n1)), m1 = fmaxf(fmaf(s[k][2], u0, n0), fmaf(s[k][3], u1, n1));
                                    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 1));
                                    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
                                    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 2));
                                    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 2));
                                    const int key = k * 16 + r + 8 * t;
                                    if (t < 2 && key < left)
                                        scores[long(mine) * BLK + tile * 16 + key] = t ? m1 : m0;
                                }
                            }
                            if (left < STEP * 16) {
#pragma unroll
                                for (int k = 0; k < STEP; k++) {
                                    if (k * 16 + r >= left) s[k][0] = s[k][1] = 0.0f;
                                    if (k * 16 + r + 8 >= left) s[k][2] = s[k][3] = 0.0f;
                                    rows[k].mask(lane, left - k * 16);
                                }
                            }
                            float w[STEP][4], top = 0.0f;
#pragma unroll
                            for (int k = 0; k < STEP; k++) {
                                flagged |= rows[k].large();
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    s[k][e] = relu_nan(s[k][e]);
                                    w[k][e] = s[k][e] * ((e & 1) ? f1 : f0) * s[k][e];
                                    top = fmaxf(top, w[k][e]);
                                }
                            }
                            bool wide = false;
                            if (__any_sync(0xffffffffu, top > KD_LIMIT || flagged)) {
#pragma unroll
                                for (int k = 0; k < STEP; k++) wide |= rows[k].wide();
                                wide = __any_sync(0xffffffffu, wide);
                                if (__any_sync(0xffffffffu, top > KD_LIMIT)) {
                                    // (a handful of times a warp) new factors: the tiles' largest weight of a head at most 2^target
                                    float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
                                    for (int k = 0; k < STEP; k++) {
                                        m0 = fmaxf(m0, fmaxf(s[k][0], s[k][2]));
                                        m1 = fmaxf(m1, fmaxf(s[k][1], s[k][3]));
                                    }
#pragma unroll
                                    for (int o = 4; o < 32; o <<= 1) {
                                        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
                                        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
                                    }
                                    // m < 2^(e + 1), so m^2 2^(target - 2 (e + 1)) < 2^target
                                    const int e0 = int(__float_as_uint(m0) >> 23) - 126, e1 = int(__float_as_uint(m1) >> 23) - 126;
                                    const float nf0 = m0 * f0 * m0 > KD_LIMIT ? pow2_biased(min(max(127 + KD_TARGET - 2 * e0, 1), 254)) : f0;
                                    const float nf1 = m1 * f1 * m1 > KD_LIMIT ? pow2_biased(min(max(127 + KD_TARGET - 2 * e1, 1), 254)) : f1;
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
#pragma unroll
                                    for (int k = 0; k < STEP; k++)
#pragma unroll
                                        for (int e = 0; e < 4; e++) w[k][e] = s[k][e] * ((e & 1) ? f1 : f0) * s[k][e];
                                }
                            }
#pragma unroll
                            for (int k = 0; k < STEP; k++) {
                                ps0 += w[k][0] + w[k][2];
                                ps1 += w[k][1] + w[k][3];
                                if (!wide) kv4_tile_values<DT>(kaddr + KV4_SIDE + k * 16 * KV4_ROW, rows[k], w[k], O);
                                else kv4_tile_values_wide(kaddr + KV4_SIDE + k * 16 * KV4_ROW, rows[k], w[k], O);
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&empty[st]);
                    st += GROUPS;
                    if (st >= STAGES) {
                        st -= STAGES;
                        phase ^= 1;
                    }
                }
                // ---- the warp's sums of the piece, in units of the weights themselves, once the helpers have read its last ones
                if (ok && given > 0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(p.ctl.wait_cycles, &taken[group], (given - 1) & 1));
                if (!ok) {
                    fail(ERR_WAIT_FULL);
                    break;
                }
                given++;
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    ps0 += __shfl_xor_sync(0xffffffffu, ps0, o);
                    ps1 += __shfl_xor_sync(0xffffffffu, ps1, o);
                }
                // w = w' / f x (the query's power of two x 2^20)^2 / 128, the powers of two multiplied one by one
                const int lane_s = here(lane), rs = lane_s >> 2, ts = lane_s & 3;
                const float q0 = pow2_biased(max(slot.sq.expo[2 * ts], 1)), q1 = pow2_biased(max(slot.sq.expo[2 * ts + 1], 1));
                const float i0 = (1.0f / 128.0f / KV4_SUBNORMAL / KV4_SUBNORMAL) / f0, i1 = (1.0f / 128.0f / KV4_SUBNORMAL / KV4_SUBNORMAL) / f1;
                float* row0 = sums + (warp * 8 + 2 * ts) * KD_SUM;
                float* row1 = row0 + KD_SUM;
                if (2 * ts < p.G) {
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int d = kv4_dim_of(k, rs);
                        row0[d] = O[k][0] * i0 * q0 * q0;
                        row1[d] = O[k][1] * i1 * q1 * q1;
                        row0[d + 2] = O[k][2] * i0 * q0 * q0;
                        row1[d + 2] = O[k][3] * i1 * q1 * q1;
                    }
                    if (rs == 0) {
                        row0[HD] = ps0 * i0 * q0 * q0;
                        row1[HD] = ps1 * i1 * q1 * q1;
                    }
                }
            }
            if (CL) break;                                          // (the cluster's CTAs meet below, all warps)
            piece0 += n;
            __syncwarp();
            if (lane == 0) mbar_arrive(&summed[j % BUFS]);
        }
    }

    trace_last(p.ctl.trace, 2);
    // Every page that was requested has been waited for, unless a wait gave up - then wait (bounded) for what is in flight.
    __syncthreads();
    if (s_failed && tid == 0) {
        for (int i = max(0, s_issued - STAGES); i < s_issued; i++)
            if (!mbar_wait_bounded(p.ctl.wait_cycles, &full[i % STAGES], (i / STAGES) & 1)) atomicExch(p.ctl.err, ERR_WAIT_DRAIN);
    }
    if (CL) {
        // every range's rows go, head by head, to the CTA that finishes the head; it adds them in range order
        constexpr int THREADS = (NCONS + 1 + KD_HELPERS) * 32;
        const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
        const float sink = sqrtf(float(HD));
        float* inbox = sums + NCONS * 8 * KD_SUM;
        const int own = (p.G + p.nsplit - 1) / p.nsplit;
        cluster_wait();
        for (int idx = tid; idx < p.G * HD; idx += THREADS) {
            const int hh = idx >> 7, d = idx & 127;
            float num = 0.0f, den = 0.0f;
#pragma unroll
            for (int w = 0; w < NCONS; w++) {
                num += sums[(w * 8 + hh) * KD_SUM + d];
                den += sums[(w * 8 + hh) * KD_SUM + HD];
            }
            const uint32_t row = cluster_map(smem_u32(inbox + (split * own + hh / p.nsplit) * KD_PART), uint32_t(hh % p.nsplit));
            cluster_st_f32(row + uint32_t(d) * 4u, num);
            if (d == 0) cluster_st_f32(row + HD * 4, den);
        }
        cluster_arrive();
        cluster_wait();
        for (int idx = tid; idx < own * HD; idx += THREADS) {
            const int slot = idx >> 7, d = idx & 127, hh = split + slot * p.nsplit;
            if (hh < p.G) {
                float num = 0.0f, den = sink;
                for (int k = 0; k < p.nsplit; k++) {
                    const float* row = inbox + (k * own + slot) * KD_PART;
                    den += row[HD];
                    num += row[d];
                }
                Act<DT>::store(p.o, size_t(b) * p.o_stride + size_t(kvh * p.G + hh) * HD + d, num / den);
            }
        }
    }
    trace_last(p.ctl.trace, 3);
}

// Adds the pieces of the units that the runs of a launch cut and writes their rows, launched behind the runs: one CTA a unit and
// head. What it costs is the latency of its loads, 1.2 to 2.8 microseconds for each round of them: four warps take every fourth
// piece, four loads in flight each, so that up to 16 pieces are one round, and add up through shared memory in a fixed order.
template <int DT>
__global__ void __launch_bounds__(128) kv4_decode_join_kernel(const __grid_constant__ Kv4DecodeParams p) {
    __shared__ float4 others[3][32];
    __shared__ float dens[3];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hh = blockIdx.x, unit = blockIdx.y, b = unit / p.n_kv_heads, kvh = unit % p.n_kv_heads;
    trace_first(p.ctl.trace, 0);
    unsigned before = 0, sum = 0;
    for (int i = lane; i < p.batch; i += 32) {
        const unsigned n = kd_cost(kd_pages(p.seq_lens, i));
        sum += n;
        if (i < b) before += n;
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    before = __reduce_add_sync(0xffffffffu, before);
    const int pages = kd_pages(p.seq_lens, b);
    const KdRuns runs(sum * p.n_kv_heads, p.n_runs);
    const unsigned x = before * p.n_kv_heads + unsigned(kvh) * kd_cost(pages);
    const int lo = int(runs.run_of(x + KD_UNIT_COST)), hi = int(runs.run_of(x + KD_UNIT_COST + pages - 1));
    // (run lo may begin inside the unit, or with the end of one before it, which is a piece: pages come last in a unit's cost)
    const int first_slot = runs.start_of(lo) >= x ? 2 * lo : 2 * lo + 1;
    // (every CTA waits, one with nothing to add too: the launch behind this one takes its end for the end of the runs)
    pdl_wait();
    pdl_launch_dependents();
    trace_first(p.ctl.trace, 1);
    if (pages == 0 || lo == hi) return;
    float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float den = 0.0f;
    for (int k = lo + warp; k <= hi; k += 16) {
        float4 v[4];
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int piece = min(k + 4 * j, hi);   // (behind the last one: loaded again and not added)
            const float* row = p.partials + (size_t(piece == lo ? first_slot : 2 * piece) * p.G + hh) * KD_PART;
            v[j] = __ldcg(reinterpret_cast<const float4*>(row) + lane);
            e[j] = __ldcg(row + HD);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool add = k + 4 * j <= hi;
            num.x += add ? v[j].x : 0.0f;
            num.y += add ? v[j].y : 0.0f;
            num.z += add ? v[j].z : 0.0f;
            num.w += add ? v[j].w : 0.0f;
            den += add ? e[j] : 0.0f;
        }
    }
    if (warp > 0) {
        others[warp - 1][lane] = num;
        if (lane == 0) dens[warp - 1] = den;
    }
    __syncthreads();
    if (warp > 0) return;
    den += sqrtf(float(HD));
#pragma unroll
    for (int w = 0; w < 3; w++) {
        const float4 v = others[w][lane];
        num.x += v.x;
        num.y += v.y;
        num.z += v.z;
        num.w += v.w;
        den += dens[w];
    }
    const size_t at = size_t(b) * p.o_stride + size_t(kvh * p.G + hh) * HD + 4 * lane;
    Act<DT>::store(p.o, at, num.x / den);
    Act<DT>::store(p.o, at + 1, num.y / den);
    Act<DT>::store(p.o, at + 2, num.z / den);
    Act<DT>::store(p.o, at + 3, num.w / den);
    trace_last(p.ctl.trace, 3);
}

// A CTA an SM: 12 consumer warps (at 128 registers the SM holds no more beside producer and helpers), four to a page, nine pages in
// flight. A cluster's CTA:
// one tile a warp, so that a page or two are done soonest.
template <bool CL> struct KdShape {
    static constexpr int ncons = CL ? 8 : 12, wpg = CL ? 8 : 4, stages = CL ? 4 : 9;
};

static bool use_pdl() {
    static const bool on = []() { const char* e = getenv("EMBLA_NO_PDL"); return !(e && e[0] == '1'); }();
    return on;
}

template <int DT, bool SCORES, bool CL>
static EmblaStatus launch_kv4_decode(EmblaAttn* ctx, const EmblaKVPool* pool, const Kv4DecodeParams& p, int batch, dim3 grid, cudaStream_t s) {
    using Shape = KdShape<CL>;
    auto kern = kv4_decode_kernel<DT, SCORES, Shape::ncons, Shape::wpg, Shape::stages, CL>;
    constexpr size_t fixed = kd_smem(Shape::ncons, Shape::stages, CL);
    const size_t smem = fixed + (CL ? kd_inbox_rows(p.nsplit, p.G) * KD_PART * 4 : 0);
    static bool configured[64] = {};   // per instantiation and device
    if (!configured[ctx->device & 63]) {
        // (the largest inbox: 7 ranges of 8 heads, two each)
        EMBLA_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(fixed + (CL ? 14 * KD_PART * 4 : 0))));
        configured[ctx->device & 63] = true;
    }
    EMBLA_CUDA_TRY(launch_kernel_cluster(ctx->pdl, CL ? p.nsplit : 1, kern, grid, dim3((Shape::ncons + 1 + KD_HELPERS) * 32), smem, s, pool->tmap_codes, p));
    if (!CL && p.n_runs > 1) {
        Kv4DecodeParams pj = p;
        pj.ctl = kernel_ctl(ctx);
        EMBLA_CUDA_TRY(launch_kernel(use_pdl(), kv4_decode_join_kernel<DT>, dim3(p.G, unsigned(batch) * p.n_kv_heads), dim3(128), 0, s, pj));
    }
    EMBLA_CUDA_TRY(cudaGetLastError());
    return EMBLA_OK;
}

// How many clusters of `ns` CTAs of the cluster form the GPU holds at once (all forms of it are alike in what they need).
static long kd_clusters_at_once(const EmblaAttn* ctx, int ns) {
    static int known[64][KD_MAX_CLUSTER + 1] = {};   // per device and size; 0: not asked yet, -1: none
    int& n = known[ctx->device & 63][ns];
    if (n == 0) {
        using Shape = KdShape<true>;
        auto kern = kv4_decode_kernel<EMBLA_BF16, false, Shape::ncons, Shape::wpg, Shape::stages, true>;
        const size_t smem = kd_smem(Shape::ncons, Shape::stages, true) + 14 * KD_PART * 4;
        int got = 0;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) == cudaSuccess) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(ns);
            cfg.blockDim = dim3((Shape::ncons + 1 + KD_HELPERS) * 32);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute at;
            at.id = cudaLaunchAttributeClusterDimension;
            at.val.clusterDim.x = unsigned(ns);
            at.val.clusterDim.y = 1;
            at.val.clusterDim.z = 1;
            cfg.attrs = &at;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&got, kern, &cfg) != cudaSuccess) got = 0;
        }
        (void)cudaGetLastError();
        n = got > 0 ? got : -1;
    }
    return n;
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
    p.batch = view->batch;
    p.prenormed = q->prenormed;
    p.ng = q->ng;
    const long units = long(view->batch) * pool->n_kv_heads, pages = (max_len + BLK - 1) / BLK;
    if (units * (pages + KD_UNIT_COST) > 0x7fffffffL || units > 0xffff)
        EMBLA_FAIL(EMBLA_BAD_ARG, "embla_attn_full_decode: %d sequences of up to %d keys are too many pages", view->batch, max_len);
    // Two ways, by what they measured, in hundredths of a microsecond: clusters, all at once, 570 + 62 a page of a range (one
    // sequence of 1000 keys 5.6 us when it was fitted, 6.6 with kv4_tile_values_wide in the kernel, of 8192 10.5); runs, 1000 + 50 a page or unit cost of a run (10.0 us at the shortest, 64 sequences
    // of 1000 keys 20.0, 8 of 32768 37.8). The ranges of a unit are as many as let all clusters be resident (a GPC may hold one cluster of
    // 8 such CTAs and not two) and no longer than 8 pages: longer ones are read at the pace of the longest sequence, where runs
    // even uneven lengths out. Runs: the scratch holds two pieces of each (embla_attn_create makes it 8 slots an SM and more).
    const long cost = units * (pages + KD_UNIT_COST), most = (cost + KD_MIN_RUN - 1) / KD_MIN_RUN;
    p.n_runs = int(most < ctx->sm_count ? most : ctx->sm_count);
    long best = 1000 + 50 * ((cost + p.n_runs - 1) / p.n_runs);
    bool cluster = false;
    dim3 grid(p.n_runs);
    for (int ns = 1; ns <= KD_MAX_CLUSTER && ns <= pages; ns++) {
        const long c = 570 + 62 * ((pages + ns - 1) / ns);
        if (c < best && (pages + ns - 1) / ns <= 8 && units <= kd_clusters_at_once(ctx, ns)) {
            best = c;
            cluster = true;
            p.nsplit = ns;
            grid = dim3(ns, pool->n_kv_heads, view->batch);
        }
    }
    const bool bf = ctx->cfg.act_dtype == EMBLA_BF16;
#define EMBLA_KD(DT, SC) (cluster ? launch_kv4_decode<DT, SC, true>(ctx, pool, p, view->batch, grid, stream) \
                                  : launch_kv4_decode<DT, SC, false>(ctx, pool, p, view->batch, grid, stream))
    if (scores_dev) return bf ? EMBLA_KD(EMBLA_BF16, true) : EMBLA_KD(EMBLA_F16, true);
    return bf ? EMBLA_KD(EMBLA_BF16, false) : EMBLA_KD(EMBLA_F16, false);
#undef EMBLA_KD
}

}  // namespace embla
