"""The 4-bit cache as a model uses it: layers in a stack, chunks then single tokens, forked sequences, captured graphs, streams."""
import numpy as np
import pytest

from oracle import oracle as orc
from tests import kv4, util

pytestmark = pytest.mark.gpu


def _stack(kinds, batch, ctx, dtype=orc.F16, Hq=8, Hkv=2, seed=0, fill=True, **kw):
    import torch
    from embla_metal_b200 import attn, stack as stk
    st = stk.DecodeStack(kinds, batch, ctx, n_q_heads=Hq, n_kv_heads=Hkv, act_dtype=dtype, window=128, ring=1024, kv_dtype=attn.KV_INT4, **kw)
    if fill:
        st.fill_random(seed)
    st.qkv.copy_(torch.randn(st.qkv.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed + 1)).to(st.dtype))
    return st


def _full_rows(st, li, b, n):
    """Values of layer li's keys and values of sequence b, [Hkv, n, 128] float64."""
    from embla_metal_b200 import stack as stk
    slot = sum(1 for k in st.kinds[:li] if k == stk.FULL)
    pages = st.full_pool.raw()[st.table[b, :(n + 127) // 128].long(), slot].cpu().numpy().transpose(1, 0, 2)
    k, v = kv4.page_values(pages)
    return k.reshape(st.Hkv, -1, 128)[:, :n], v.reshape(st.Hkv, -1, 128)[:, :n]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("pos", [[0, 127, 128], [1200, 1151, 40], [1152, 700, 1999]])
def test_step_of_full_and_shared_sparse_layers(dtype, pos):
    """[full (scores, selection), sparse over its cache, sliding, full]: the appended rows, then each layer against the formulas on
    the very pages the step left behind."""
    import torch
    from embla_metal_b200 import attn, stack as stk
    dt = orc.F16 if dtype == "f16" else orc.BF16
    st = _stack([stk.FULL, stk.SPARSE_SHARED, stk.SLIDING, stk.FULL], 3, 2048, dt, norm_k=True)
    st.set_positions(pos)
    before = st.full_pool.raw().clone()
    st.step()
    st.ctx.check()
    G = st.Hq // st.Hkv
    width = st.Hq * 128
    qkv = orc.from_bits(util.act_bits(st.qkv), dt).astype(np.float64)
    o = orc.from_bits(util.act_bits(st.o), dt).astype(np.float64)
    changed = (st.full_pool.raw() != before).flatten(2).any(2).nonzero().tolist()
    assert sorted(changed) == sorted([int(st.table[b, p // 128]), l] for b, p in enumerate(pos) for l in range(2))
    for li, slot in ((0, 0), (3, 1)):
        for b, p in enumerate(pos):
            k, v = _full_rows(st, li, b, p + 1)
            for h in range(st.Hkv):
                raw_k = qkv[li, b, width + h * 128:width + (h + 1) * 128]
                raw_v = qkv[li, b, width + (st.Hkv + h) * 128:width + (st.Hkv + h + 1) * 128]
                nk = orc.from_bits(orc.to_bits(raw_k.astype(np.float32) * kv4.norm_rows32(raw_k), dt), dt)
                assert np.array_equal(k[h, p], kv4.values(*kv4.quantise(nk)))
                assert np.array_equal(v[h, p], kv4.values(*kv4.quantise(raw_v)))
                q = qkv[li, b, h * G * 128:(h + 1) * G * 128].reshape(G, 128)
                want, bound = kv4.relu2(q, k[h], v[h], np.ones((G, p + 1), bool), kv4.U16[dtype])
                got = o[li, b, h * G * 128:(h + 1) * G * 128].reshape(G, 128)
                assert (np.abs(got - want) <= bound).all(), (li, b, h)
    # the sparse layer attends every key up to 1152, then the 1024 best of the first full layer's scores and the 128 latest. The
    # scores once more, for the rows that the selection takes of them; that those are the best ones is checked against the formula.
    sc = torch.zeros(3, st.Hkv, 2048, device="cuda")
    idx = torch.zeros(3, st.Hkv, 1152, dtype=torch.int32, device="cuda")
    st.ctx.full_decode(st.full_pool, st.table, st.seq_lens, 0, st.qkv[0], torch.zeros_like(st.o[0]), scores=sc, max_seq_len=st.max_seq_len)
    st.ctx.select_keys(sc, st.seq_lens, idx, max_seq_len=st.max_seq_len)
    st.ctx.check()
    for b, p in enumerate(pos):
        k, v = _full_rows(st, 0, b, p + 1)
        for h in range(st.Hkv):
            q0 = qkv[0, b, h * G * 128:(h + 1) * G * 128].reshape(G, 128)
            q1 = qkv[1, b, h * G * 128:(h + 1) * G * 128].reshape(G, 128)
            at = np.arange(p + 1)
            if p + 1 > 1152:
                at = idx[b, h].cpu().numpy()
                s = (q0 @ k[h].T).max(0)
                err = kv4.DOT * (np.abs(q0) @ np.abs(k[h]).T).max()
                assert len(set(at.tolist())) == 1152 and np.array_equal(at[1024:], np.arange(p + 1 - 128, p + 1))
                assert s[at[:1024]].min() >= np.sort(s[:p + 1 - 128])[-1024] - 2 * err
            want, bound = kv4.softmax(q1, k[h][at], v[h][at], kv4.U16[dtype])
            got = o[1, b, h * G * 128:(h + 1) * G * 128].reshape(G, 128)
            assert (np.abs(got - want) <= bound).all(), (b, h)
    st.close()


@pytest.mark.parametrize("no_early", ["0", "1"])
def test_step_equals_the_calls_one_by_one(no_early, monkeypatch):
    """A step's launches overlap (dependent launch, pages fetched ahead): the same bits as append and attention called apart."""
    import torch
    from embla_metal_b200 import attn, stack as stk
    monkeypatch.setenv("EMBLA_NO_EARLY", no_early)
    kinds = [stk.FULL] * 4
    a = _stack(kinds, 5, 6000, seed=3)
    a.set_positions([5000, 17, 128, 5999, 2047])
    pages = a.full_pool.raw().clone()
    for _ in range(3):
        a.full_pool.raw().copy_(pages)
        a.o.zero_()
        a.step()
        a.ctx.check()
        after, o = a.full_pool.raw().clone(), a.o.clone()
        a.full_pool.raw().copy_(pages)
        one = torch.zeros_like(a.o)
        w, kw = a.Hq * 128, a.Hkv * 128
        for li in range(4):
            row = a.qkv[li]
            a.ctx.kv_append(a.full_pool, a.table, li, a.pos, row[:, None, w:w + kw], row[:, None, w + kw:w + 2 * kw], norm_k=False)
            a.ctx.full_decode(a.full_pool, a.table, a.seq_lens, li, row, one[li], max_seq_len=a.max_seq_len)
        a.ctx.check()
        assert torch.equal(after, a.full_pool.raw()) and torch.equal(o, one)
    step = torch.zeros_like(a.o[0])
    a.full_pool.raw().copy_(pages)
    row = a.qkv[1]
    a.ctx.full_step(a.full_pool, a.table, a.seq_lens, 1, row, row[:, w:w + kw], row[:, w + kw:w + 2 * kw], step, max_seq_len=a.max_seq_len,
                    norm_k=False)
    a.ctx.check()
    assert torch.equal(step, one[1])
    a.close()


def test_chunk_then_tokens_against_tokens_alone():
    """A 150-token chunk through [full, sliding, full] leaves the bytes that 150 steps leave, and outputs within their roundings."""
    import torch
    from embla_metal_b200 import stack as stk
    kinds = [stk.FULL, stk.SLIDING, stk.FULL]
    T = 150
    a, b = (_stack(kinds, 2, 512, orc.BF16, seed=5, fill=False, norm_k=True) for _ in range(2))
    g = torch.Generator("cuda").manual_seed(9)
    qkv = torch.randn(3, 2, T, a.qkv_width, device="cuda", generator=g).to(a.dtype)
    o = torch.zeros(3, 2, T, a.o_width, dtype=a.dtype, device="cuda")
    a.prefill_chunk(qkv, o, torch.zeros(2, dtype=torch.int32, device="cuda"), max_seq_len=T)
    a.ctx.check()
    for t in range(T):
        b.qkv.copy_(qkv[:, :, t])
        b.set_positions(t)
        b.step()
        # two bf16 outputs of the same sums: half a step each of 2^-8, and the chunk's fp16 products (2^-11 on keys, values and
        # weights, the weight a square: 6 x 2^-11 of the sum of magnitudes, here under 4 in size)
        d = (o[:, :, t].double() - b.o.double()).abs()
        assert (d <= b.o.double().abs() * 2.0 ** -7 + 6 * 2.0 ** -11 * 4).all(), t
    b.ctx.check()
    assert torch.equal(a.full_pool.raw(), b.full_pool.raw())
    a.close()
    b.close()


@pytest.mark.parametrize("n", [1, 127, 128, 300, 1300])
def test_fork_goes_on_like_a_copy(n):
    import torch
    from embla_metal_b200 import stack as stk
    kinds = [stk.FULL, stk.SPARSE_SHARED, stk.SPARSE, stk.SLIDING]
    st = _stack(kinds, 3, 2048, seed=7)
    whole = _stack(kinds, 3, 2048, seed=7)
    for s in (st, whole):
        s.set_positions([n - 1, 5, 5])
    st.fork(0, 2)
    # the copy to compare with: every block of sequence 0 copied whole into sequence 2's own
    for pool in (whole.full_pool, whole.sparse_pool):
        pool.raw()[2 * whole.npages:] = pool.raw()[:whole.npages]
    for r in whole.rings:
        r.k[2].copy_(r.k[0])
        r.v[2].copy_(r.v[0])
    whole.set_positions([n - 1, 5, n - 1])
    full = n // 128
    assert torch.equal(st.table[2, :full], st.table[0, :full]) and int(st.seq_lens[2]) == n
    assert (st.table[2, full:] == torch.arange(2 * st.npages + full, 3 * st.npages, device="cuda")).all()
    for i in range(3):                    # both go on, with tokens of their own
        pos = [n + i, 6 + i, n + i]
        q = torch.randn(st.qkv.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(i)).to(st.dtype)
        for s in (st, whole):
            s.qkv.copy_(q)
            s.set_positions(pos)
            s.step()
            s.ctx.check()
        assert torch.equal(st.o, whole.o), i
    with pytest.raises(ValueError):
        st.fork(1, 1)
    with pytest.raises(ValueError):
        st.fork(0, 3)
    if full:
        with pytest.raises(ValueError):   # sequence 2 shares blocks of sequence 0
            st.fork(1, 0)
    st.close()
    whole.close()


def test_captured_step_replays_with_other_positions():
    import torch
    from embla_metal_b200 import stack as stk
    st = _stack([stk.FULL, stk.SPARSE_SHARED, stk.FULL], 4, 4096, seed=11)
    ref = _stack([stk.FULL, stk.SPARSE_SHARED, stk.FULL], 4, 4096, seed=11)
    for s in (st, ref):
        s.set_positions([4000, 1152, 3, 2500])
        s.max_seq_len = 4096
    s0 = torch.cuda.Stream()
    with torch.cuda.stream(s0):
        st.step()
        s0.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s0):
            st.step()
        for i in range(4):
            pos = [4000 + i, 1152 + 300 * i, 3 + i, 2500 - 700 * i]
            q = torch.randn(st.qkv.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(20 + i)).to(st.dtype)
            for s in (st, ref):
                s.qkv.copy_(q)
                s.set_positions(pos)
                s.max_seq_len = 4096
            graph.replay()
            ref.step()
            s0.synchronize()
            assert torch.equal(st.o, ref.o), i
        st.ctx.check()
        ref.ctx.check()
    del graph
    st.close()
    ref.close()


def test_two_contexts_on_two_streams():
    """Contexts of their own on streams of their own, working at the same time over one pool (read only)."""
    import torch
    from embla_metal_b200 import attn
    from tests.test_kv4_gpu import _queries, _setup
    lens = [3000, 50, 1500, 0]
    rng, ctx, pool, table, k, v = _setup("f16", 8, 2, lens, 31)
    other = attn.Attention(8, 2, attn.F16, 4, 4096)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = [_queries(rng, 4, 8, "f16", 0)[0] for _ in range(2)]
    want = []
    for c, q in zip((ctx, other), qs):
        o = torch.zeros(4, 1024, dtype=torch.float16, device="cuda")
        c.full_decode(pool, table, ln, 1, q, o)
        want.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.zeros(20, 4, 1024, dtype=torch.float16, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(20):
        for c, q, s, o in zip((ctx, other), qs, streams, outs):
            with torch.cuda.stream(s):
                c.full_decode(pool, table, ln, 1, q, o[i])
    torch.cuda.synchronize()
    for c in (ctx, other):
        c.check()
    for o, w in zip(outs, want):
        assert all(torch.equal(o[i], w) for i in range(20))


@pytest.mark.parametrize("batch,n", [(1, 3000), (6, 9000)])
def test_a_stalled_producer_is_reported_and_the_next_call_is_right(batch, n):
    """The consumers' waits run out (short limit, the producer stops at page 2 of its run), the status says so, and the context
    works on: in the cluster form and in the form with runs."""
    import torch
    from embla_metal_b200 import attn
    from tests.test_kv4_gpu import _queries, _setup
    rng, ctx, pool, table, k, v = _setup("f16", 8, 4, [n] * batch, 41)
    ln = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    q = _queries(rng, batch, 8, "f16", 0)[0]
    good, o = (torch.zeros(batch, 1024, dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.full_decode(pool, table, ln, 1, q, good)
    ctx.check()
    ctx.set_wait_limit(200000)
    ctx.inject_stall(2)
    ctx.full_decode(pool, table, ln, 1, q, o)
    with pytest.raises(attn.EmblaError) as e:
        ctx.check()
    assert e.value.status == attn.TIMEOUT
    ctx.inject_stall(None)
    ctx.set_wait_limit(1 << 30)
    ctx.full_decode(pool, table, ln, 1, q, o)
    ctx.check()
    assert torch.equal(o, good)


def test_shared_blocks_are_not_written_and_are_given_back():
    import torch
    from embla_metal_b200 import stack as stk
    st = _stack([stk.FULL, stk.SPARSE], 4, 1024, seed=8)
    st.set_positions([299, 5, 5, 5])
    st.fork(0, 1)
    st.fork(1, 2)                          # shares blocks of sequence 0 through sequence 1, and has its own last one
    for pos in ([255, 300, 300, 5], [300, 0, 300, 5], [300, 300, 255, 5]):
        with pytest.raises(ValueError):
            st.set_positions(pos)
    st.set_positions([300, 256, 299, 0])   # inside the blocks that each has to itself
    for b in (0, 4, -1):
        with pytest.raises(ValueError):
            st.restart(b)                  # others share its blocks; no such sequence
    before = st.full_pool.raw()[:2].clone()
    st.restart(1)
    st.set_positions([300, 0, 300, 0])
    st.qkv.normal_()
    st.step()
    st.ctx.check()
    assert torch.equal(st.full_pool.raw()[:2], before)
    assert st.table[1].tolist() == list(range(st.npages, 2 * st.npages))
    with pytest.raises(ValueError):
        st.restart(0)                      # sequence 2 still does
    st.restart(2)
    st.restart(0)
    st.set_positions(0)
    st.close()
