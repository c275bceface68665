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
