"""Long contexts over the 4-bit cache, piece by piece: each call is cut among CTAs and clusters by its size, and joined. The elementwise bounds of
kv4.py add the keys' roundings up, which at these lengths leaves room for a page; here a lost page, tile or key is the whole output, and
outputs are compared as a whole."""
import numpy as np
import pytest

from tests import kv4
from tests.test_kv4_gpu import DT, _act, _bits, _out, _queries, _setup, _val

pytestmark = pytest.mark.gpu

SINK = np.sqrt(128.0)


def _spots(n, rng):
    """Positions at the borders of pages and tiles, at both ends, and anywhere."""
    at = [0, 15, 16, 127, 128, n - 1, n - 2, (n - 1) // 128 * 128, (n - 1) // 16 * 16] + rng.integers(0, n, 7).tolist()
    return sorted({min(max(int(t), 0), n - 1) for t in at})


class _OneValue:
    """A cache whose values are zeros but for one key a sequence, which the queries weigh."""

    def __init__(self, dtype, Hq, Hkv, lens, seed):
        import torch
        self.torch, self.dtype, self.lens, self.G = torch, dtype, lens, Hq // Hkv
        self.rng, self.ctx, self.pool, self.table, self.k, _ = _setup(dtype, Hq, Hkv, lens, seed)
        raw = self.pool.raw()
        for b, n in enumerate(lens):                       # zero codes: whatever the scales, but for rows behind the last key
            raw[self.table[b, :(n + 127) // 128].long(), 1, :, kv4.SIDE:2 * kv4.SIDE] = 0
        self.full = [n for n in lens]

    def rows(self, at, k, v):
        """k, v [B, Hkv, 128] at positions `at`, as the cache keeps them."""
        t = self.torch
        kb, vb = _bits(k, self.dtype), _bits(v, self.dtype)
        flat = lambda x: _act(x.reshape(len(self.lens), 1, -1), self.dtype)
        self.ctx.kv_append(self.pool, self.table, 1, t.tensor(at, dtype=t.int32, device="cuda"), flat(kb), flat(vb), norm_k=False)
        return [kv4.values(*kv4.quantise(_val(x, self.dtype))) for x in (kb, vb)]


def _agree(got, want, rel, what):
    """Within `rel` of the row's largest output, and not zero where that is not."""
    top = np.abs(want).max(-1, keepdims=True)
    assert np.isfinite(got).all(), what
    worst = (np.abs(got - want) / top).max()
    assert worst <= rel, f"{what}: off by {worst:.3e} of the row's largest"


# a weight: its key's dot (2 x 2^-11 at most where the key is fp16, squared: 4), its own roundings (2), the value's (1), then the sum's and the
# output's own: 8 x 2^-11 and the output's half step, for all forms
REL = {d: 8 * 2.0 ** -11 + kv4.U16[d] for d in kv4.U16}


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scores", [False, True])
@pytest.mark.parametrize("Hq,Hkv,lens", [(8, 2, [3000]), (8, 4, [20001]), (6, 2, [9001, 5000, 130, 1, 700, 9000, 1280, 4097, 128, 127, 17]),
                                         (16, 4, [2049] * 40)])
def test_full_decode_has_every_key(dtype, scores, Hq, Hkv, lens):
    t = _OneValue(dtype, Hq, Hkv, lens, 3)
    torch, B = t.torch, len(lens)
    q, qv, _ = _queries(t.rng, B, Hq, dtype, 0)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qg = qv.reshape(B, Hkv, t.G, 128)
    weights = [np.maximum(np.einsum("hgd,hnd->hgn", qg[b], t.k[b]) / SINK, 0) ** 2 for b in range(B)]
    spots = [_spots(n, t.rng) for n in lens]
    sc = torch.zeros(B, Hkv, t.table.shape[1] * 128, device="cuda") if scores else None
    key, zero = qg.mean(2) * t.G ** 0.5, np.zeros((B, Hkv, 128))
    for i in range(max(len(s) for s in spots)):
        at = [s[i % len(s)] for s in spots]
        k, v = t.rows(at, key, t.rng.standard_normal((B, Hkv, 128)))
        o = torch.zeros(B, Hq * 128, dtype=t.ctx.torch_dtype, device="cuda")
        t.ctx.full_decode(t.pool, t.table, ln, 1, q, o, scores=sc)
        t.ctx.check()
        w = np.maximum(np.einsum("bhgd,bhd->bhg", qg, k) / SINK, 0) ** 2
        den = SINK + w + np.stack([weights[b].sum(-1) - weights[b][:, :, at[b]] for b in range(B)])
        _agree(_out(o, dtype).reshape(B, Hkv, t.G, 128), (w / den)[..., None] * v[:, :, None], REL[dtype], f"positions {at}")
        for b in range(B):                                 # back to what the weights were taken of, its value zero
            weights[b][:, :, at[b]] = w[b]
        t.rows(at, key, zero)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,lens", [(8, 2, [1152, 1000, 129, 1]), (4, 4, [1151] * 64), (8, 1, [5000])])
def test_sparse_decode_has_every_row(dtype, Hq, Hkv, lens):
    t = _OneValue(dtype, Hq, Hkv, lens, 5)
    torch, B = t.torch, len(lens)
    q, qv, _ = _queries(t.rng, B, Hq, dtype, 0)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qg = qv.reshape(B, Hkv, t.G, 128)
    idx = np.zeros((B, Hkv, 1152), np.int32)
    sel = []
    for b, n in enumerate(lens):
        s = np.arange(n) if n <= 1152 else np.concatenate([np.sort(t.rng.permutation(n - 128)[:1024]), np.arange(n - 128, n)])
        sel.append(s)
        if n > 1152:
            idx[b] = s
    idx = torch.from_numpy(idx).cuda()
    e = [np.exp(np.einsum("hgd,hnd->hgn", qg[b], t.k[b][:, sel[b]]) / SINK) for b in range(B)]
    spots = [_spots(len(s), t.rng) for s in sel]
    key, zero = qg.mean(2) * t.G ** 0.5, np.zeros((B, Hkv, 128))
    for i in range(max(len(s) for s in spots)):
        j = [s[i % len(s)] for s in spots]
        at = [int(sel[b][j[b]]) for b in range(B)]
        k, v = t.rows(at, key, t.rng.standard_normal((B, Hkv, 128)))
        o = torch.zeros(B, Hq * 128, dtype=t.ctx.torch_dtype, device="cuda")
        t.ctx.sparse_decode(t.pool, t.table, ln, 1, q, o, idx=idx)
        t.ctx.check()
        w = np.exp(np.einsum("bhgd,bhd->bhg", qg, k) / SINK)
        den = w + np.stack([e[b].sum(-1) - e[b][:, :, j[b]] for b in range(B)])
        _agree(_out(o, dtype).reshape(B, Hkv, t.G, 128), (w / den)[..., None] * v[:, :, None], REL[dtype], f"rows {j}")
        for b in range(B):
            e[b][:, :, j[b]] = w[b]
        t.rows(at, key, zero)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,pos0,T", [(8, 2, [6000], 64), (2, 1, [12700], 33), (8, 2, [6000], 1024), (2, 1, [12000], 700), (16, 4, [700, 663, 626], 333),
                                           (16, 2, [100, 0], 517)])
def test_full_prefill_has_every_key(dtype, Hq, Hkv, pos0, T):
    """The same key for all tokens of a chunk; those ahead of it have zeros."""
    from embla_metal_b200 import attn
    lens = [p + T for p in pos0]
    t = _OneValue(dtype, Hq, Hkv, lens, 7)
    torch, B = t.torch, len(lens)
    base = t.rng.standard_normal((B, 1, Hkv, 1, 128))
    bits = _bits((base + 0.7 * t.rng.standard_normal((B, T, Hkv, t.G, 128))).reshape(B, T, Hq * 128), dtype)
    qv = _val(bits, dtype).reshape(B, T, Hkv, t.G, 128)
    q = _act(bits, dtype)
    p0 = torch.tensor(pos0, dtype=torch.int32, device="cuda")
    seen = [np.arange(lens[b])[None] <= pos0[b] + np.arange(T)[:, None] for b in range(B)]
    weights = [np.maximum(np.einsum("thgd,hnd->thgn", qv[b], t.k[b], optimize=True) / SINK, 0) ** 2 * seen[b][:, None, None] for b in range(B)]
    spots = [_spots(n, t.rng) for n in lens]
    key, zero = base[:, 0, :, 0], np.zeros((B, Hkv, 128))
    for i in range(max(len(s) for s in spots)):
        at = [s[i % len(s)] for s in spots]
        k, v = t.rows(at, key, t.rng.standard_normal((B, Hkv, 128)))
        o = torch.zeros(B, T, Hq * 128, dtype=t.ctx.torch_dtype, device="cuda")
        attn.full_prefill(t.ctx, t.pool, t.table, 1, p0, q, o)
        t.ctx.check()
        got = _out(o, dtype).reshape(B, T, Hkv, t.G, 128)
        for b in range(B):
            w = np.maximum(np.einsum("thgd,hd->thg", qv[b], k[b]) / SINK, 0) ** 2 * seen[b][:, at[b], None, None]
            den = SINK + w + weights[b].sum(-1) - weights[b][..., at[b]]
            sees = seen[b][:, at[b]]
            assert (got[b][~sees] == 0).all()
            _agree(got[b][sees], ((w / den)[..., None] * v[b][None, :, None])[sees], REL[dtype], f"sequence {b}, position {at[b]}")
            weights[b][..., at[b]] = w
        t.rows(at, key, zero)


# ---- as a whole --------------------------------------------------------------------------------------------------
# An output is a sum of terms of either sign, so independent relative errors of its terms are relative errors of the row as a root of the mean square. A
# rounding within half a step u is 0.41 u so (uniform in the step, the number anywhere between two powers of two). Decode: a weight times a
# scale (bf16 outputs: two roundings) and the output: 0.58 x 2^-11 in fp16, 0.41 x 2^-8 in bf16; the limit is 1.2 u. A lost 16-key tile of
# 32768 keys is 2^-5.5.
def _whole(got, want, dtype, what):
    rms = np.sqrt(((got - want) ** 2).sum(-1) / (want ** 2).sum(-1))
    assert rms.max() < 1.2 * kv4.U16[dtype], f"{what}: {rms.max():.3e} of the row"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scores", [False, True])
@pytest.mark.parametrize("lens", [[32768], [20001, 32768, 31999, 12345], [6001] * 20])
@pytest.mark.parametrize("kscale", [1.0, 0.02])
def test_long_decode_as_a_whole(dtype, scores, lens, kscale):
    """(Keys of 0.02: a few of their weights' sums beside the sink, which is most of the denominator.)"""
    import torch
    Hq, Hkv = 8, 2
    rng, ctx, pool, table, k, v = _setup(dtype, Hq, Hkv, lens, 11, kscale=kscale)
    B = len(lens)
    q, qv, _ = _queries(rng, B, Hq, dtype, 0)
    o = torch.zeros(B, Hq * 128, dtype=ctx.torch_dtype, device="cuda")
    sc = torch.zeros(B, Hkv, table.shape[1] * 128, device="cuda") if scores else None
    ctx.full_decode(pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1, q, o, scores=sc)
    ctx.check()
    got = _out(o, dtype).reshape(B, Hkv, 4, 128)
    for b in range(B):
        for h in range(Hkv):
            want, _ = kv4.relu2(qv[b].reshape(Hkv, 4, 128)[h], k[b][h], v[b][h], np.ones((4, lens[b]), bool), 0.0)
            _whole(got[b, h], want, dtype, f"sequence {b}, kv head {h}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,pos0,T", [(8, 2, [6000], 1024), (2, 1, [12000], 700), (4, 1, [30000], 50), (8, 4, [5000, 4000, 3000], 130)])
def test_long_prefill_as_a_whole(dtype, Hq, Hkv, pos0, T):
    from embla_metal_b200 import attn
    import torch
    lens = [p + T for p in pos0]
    rng, ctx, pool, table, k, v = _setup(dtype, Hq, Hkv, lens, 13)
    B, G = len(lens), Hq // Hkv
    bits = _bits(rng.standard_normal((B, T, Hq * 128)), dtype)
    o = torch.zeros(B, T, Hq * 128, dtype=ctx.torch_dtype, device="cuda")
    attn.full_prefill(ctx, pool, table, 1, torch.tensor(pos0, dtype=torch.int32, device="cuda"), _act(bits, dtype), o)
    ctx.check()
    got, x = _out(o, dtype).reshape(B, T, Hq, 128), _val(bits, dtype).reshape(B, T, Hq, 128)
    for b in range(B):
        seen = np.arange(lens[b])[None] <= pos0[b] + np.arange(T)[:, None]
        for h in range(Hq):
            want, _ = kv4.relu2(x[b, :, h], k[b][h // G], v[b][h // G], seen, 0.0)
            # here keys (twice in a weight) and values are rounded as well, and relu(s) (twice) and its square: the root of 0.41^2 (4 + 1 + 4 +
            # 1 + 1) or 1.4 x 2^-11 with the output's, doubled in the limit
            rms = np.sqrt(((got[b, :, h] - want) ** 2).sum(-1) / (want ** 2).sum(-1))
            assert rms.max() < (2.0 ** -9.5 if dtype == "f16" else 1.2 * 2.0 ** -8), f"sequence {b}, head {h}: {rms.max():.3e}"
