"""The 4-bit cache where it can go wrong without a small test seeing it: rows that are not numbers at every place of a chunk, rows of every size,
and lost pieces of long contexts."""
import numpy as np
import pytest

from tests import kv4
from tests.test_kv4_gpu import DT, _act, _bits, _out, _queries, _setup, _val, _within

pytestmark = pytest.mark.gpu


# ---- what is not a number, in prefill ----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,at", [(1, 299), (40, 259), (40, 299), (40, 128), (300, 0), (300, 130), (300, 255), (300, 299)])
def test_prefill_a_key_that_is_not_a_number(dtype, T, at):
    """A NaN in one key row of the second kv head, ahead of the chunk or in it: every token from that position on, in that head, is NaN (decode
    gives the same); the tokens ahead of it and the other head are finite."""
    import torch
    from embla_metal_b200 import attn
    Hq, Hkv, n = 4, 2, 300
    rng, ctx, pool, table, k, v = _setup(dtype, Hq, Hkv, [n], at + T)
    row = torch.ones(1, 1, Hkv * 128, dtype=ctx.torch_dtype, device="cuda")
    bad = row.clone()
    bad[0, 0, 128 + 70] = float("nan")
    ctx.kv_append(pool, table, 1, torch.tensor([at], dtype=torch.int32, device="cuda"), bad, row, norm_k=False)
    p0 = n - T
    q = _act(_bits(rng.standard_normal((1, T, Hq * 128)), dtype), dtype)
    o = torch.zeros_like(q)
    attn.full_prefill(ctx, pool, table, 1, torch.tensor([p0], dtype=torch.int32, device="cuda"), q, o)
    ctx.check()
    nan = torch.isnan(o[0].float()).view(T, Hkv, -1).cpu().numpy()
    assert not nan[:, 0].any() and not torch.isinf(o).any()
    sees = np.arange(p0, n) >= at
    assert nan[sees, 1].all() and not nan[~sees, 1].any()
    d = torch.zeros(1, Hq * 128, dtype=o.dtype, device="cuda")
    ctx.full_decode(pool, table, torch.tensor([n], dtype=torch.int32, device="cuda"), 1, q[:, -1].contiguous(), d)
    ctx.check()
    assert torch.equal(torch.isnan(d), torch.isnan(o[0, -1:]))
