"""Forked sequences of a DecodeStack on the GPU, against stacks whose sequences hold copies of their own."""
import pytest

from tests.test_kv4_stack_gpu import _stack

pytestmark = pytest.mark.gpu


def _tokens(st, seed):
    import torch
    return torch.randn(st.qkv.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(st.dtype)


def _copied(st, src, dst):
    """What a fork is to equal: every block and ring of sequence src copied whole into dst's own."""
    n = st.npages
    for pool in (st.full_pool, st.sparse_pool):
        if pool is not None:
            pool.raw()[dst * n:(dst + 1) * n] = pool.raw()[src * n:(src + 1) * n]
    for r in st.rings:
        r.k[dst].copy_(r.k[src])
        r.v[dst].copy_(r.v[src])


@pytest.mark.parametrize("n", [1, 127, 128, 256, 300])
def test_a_step_straight_after_a_fork(n):
    """set_positions(n - 1), fork, and a step with tokens of their own: position n - 1 of both, in rows of their own."""
    import torch
    from embla_metal_b200 import stack as stk
    kinds = [stk.FULL, stk.SPARSE_SHARED, stk.SPARSE, stk.SLIDING]
    st, whole = (_stack(kinds, 3, 1024, seed=7) for _ in range(2))
    for s in (st, whole):
        s.set_positions([n - 1, 5, 5])
    st.fork(0, 2)
    _copied(whole, 0, 2)
    whole.set_positions([n - 1, 5, n - 1])
    for i in range(3):
        q = _tokens(st, i)
        for s in (st, whole):
            s.qkv.copy_(q)
            if i:
                s.set_positions([n - 1 + i, 5 + i, n - 1 + i])
            s.step()
            s.ctx.check()
        assert torch.equal(st.o, whole.o), i
    st.close()
    whole.close()


@pytest.mark.parametrize("kv", ["int4", "int8"])
@pytest.mark.parametrize("n", [1, 127, 128, 256, 300])
@pytest.mark.parametrize("positions", [False, True])
def test_a_fork_after_a_prompt_chunk(n, kv, positions):
    """A prompt of n tokens, forked, then steps with different tokens: bit-equal to sequences that went through the prompt themselves."""
    import torch
    from embla_metal_b200 import attn, stack as stk
    from oracle import oracle as orc
    kinds = [stk.FULL, stk.SLIDING, stk.FULL]
    both = []
    for _ in range(2):
        st = stk.DecodeStack(kinds, 3, 1024, n_q_heads=8, n_kv_heads=2, act_dtype=orc.F16, window=128, ring=1024,
                             kv_dtype=attn.KV_INT4 if kv == "int4" else attn.KV_INT8)
        st.fill_random(3)                                  # what earlier sequences left behind
        st.set_positions([700, 5, 900])
        both.append(st)
    st, whole = both
    g = torch.Generator("cuda").manual_seed(n)
    qkv = torch.randn(3, 3, n, st.qkv_width, device="cuda", generator=g).to(st.dtype)
    qkv[:, 2] = qkv[:, 0]
    o = torch.zeros(3, 3, n, st.o_width, dtype=st.dtype, device="cuda")
    pos0 = torch.zeros(3, dtype=torch.int32, device="cuda")
    whole.prefill_chunk(qkv, o, pos0, max_seq_len=n)
    qkv[:, 2].normal_()                                    # (the forked stack's sequence 2 had another prompt)
    st.prefill_chunk(qkv, o, pos0, max_seq_len=n)
    st.fork(0, 2)
    assert (st.table[2, :n // 128] == st.table[0, :n // 128]).all()
    for i in range(3):
        q = _tokens(st, i)
        for s in (st, whole):
            s.qkv.copy_(q)
            if i or positions:
                s.set_positions(n + i)
            s.step()
            s.ctx.check()
        assert torch.equal(st.o, whole.o), i
    st.close()
    whole.close()


def test_a_chunk_into_shared_blocks_is_refused():
    import torch
    from embla_metal_b200 import stack as stk
    st = _stack([stk.FULL], 2, 1024, seed=3)
    st.set_positions([299, 5])
    st.fork(0, 1)
    qkv = torch.zeros(1, 2, 4, st.qkv_width, dtype=st.dtype, device="cuda")
    o = torch.zeros(1, 2, 4, st.o_width, dtype=st.dtype, device="cuda")
    before = st.full_pool.raw().clone()
    at = lambda *p: torch.tensor(p, dtype=torch.int32, device="cuda")
    for p in (at(0, 300), at(300, 255)):
        with pytest.raises(ValueError):
            st.prefill_chunk(qkv, o, p, max_seq_len=304)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        p = at(300, 300)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(ValueError):                # (the positions cannot be looked at)
                st.prefill_chunk(qkv, o, p, max_seq_len=304)
            o.zero_()                                      # (a graph of something)
    torch.cuda.synchronize()
    assert torch.equal(st.full_pool.raw(), before)
    st.prefill_chunk(qkv, o, p, max_seq_len=304)
    st.ctx.check()
    assert torch.equal(st.full_pool.raw()[:2], before[:2])
    del graph
    st.close()
