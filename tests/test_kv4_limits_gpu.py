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


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,at,p0", [(1, 299, 299), (40, 259, 260), (40, 259, 230), (40, 128, 260), (300, 0, 0), (300, 130, 0), (300, 255, 0),
                                     (300, 299, 0), (200, 3100, 3000), (600, 3300, 2900)])
def test_prefill_a_value_that_is_not_a_number(dtype, T, at, p0):
    """A NaN in one value row of the second kv head: its group of 32 dims is NaN in every token from that position on, and in nothing else: not in the
    tokens ahead of it, whose masked weights are zeros, and not in what the rest of the row gives."""
    import torch
    from embla_metal_b200 import attn
    Hq, Hkv, n = 4, 2, p0 + T
    rng, ctx, pool, table, k, v = _setup(dtype, Hq, Hkv, [n], at + T)
    row = torch.ones(1, 1, Hkv * 128, dtype=ctx.torch_dtype, device="cuda")
    bad = row.clone()
    bad[0, 0, 128 + 70] = float("nan")
    q = _act(_bits(rng.standard_normal((1, T, Hq * 128)), dtype), dtype)
    pos = torch.tensor([p0], dtype=torch.int32, device="cuda")
    outs = []
    for x in (row, bad):
        ctx.kv_append(pool, table, 1, torch.tensor([at], dtype=torch.int32, device="cuda"), row, x, norm_k=False)
        o = torch.zeros_like(q)
        attn.full_prefill(ctx, pool, table, 1, pos, q, o)
        ctx.check()
        outs.append(o[0].float().view(T, Hkv, Hq // Hkv, 4, 32).cpu().numpy())
    want = np.zeros(outs[0].shape, bool)
    want[np.arange(p0, n) >= at, 1, :, 70 // 32] = True
    assert np.isfinite(outs[0]).all()
    assert np.array_equal(np.isnan(outs[1]), want)
    assert np.array_equal(outs[0][~want], outs[1][~want])


# ---- rows of every size, in prefill ------------------------------------------------------------------------------
def _prefill_case(dtype, Hq, Hkv, pos0, T, seed, kf=None, vf=None, qf=None, gains=False):
    """A chunk of T tokens at pos0 over rows ~ N(0, 1) times kf / vf [keys] (any size that bf16 holds), queries times qf [T]. Returns outputs [B, T, Hq,
    128], their values in 64 bits and the bounds."""
    import torch
    from embla_metal_b200 import attn
    rng = np.random.default_rng(seed)
    B, G = len(pos0), Hq // Hkv
    S = [p + T for p in pos0]
    npg = [(s + 127) // 128 for s in S]
    ctx = attn.Attention(Hq, Hkv, DT[dtype], B, max(npg) * 128)
    pool = attn.KVPool(1, Hkv, sum(npg), attn.KV_INT4)
    table = torch.zeros(B, max(npg), dtype=torch.int32, device="cuda")
    ids = rng.permutation(sum(npg)).astype(np.int32)
    k, v, at = [], [], 0
    for b in range(B):
        pages = np.zeros((Hkv, npg[b], kv4.PAGE), np.uint8)
        rows = []
        for side, f in ((0, kf), (1, vf)):
            x = rng.standard_normal((Hkv, npg[b] * 128, 128))
            if f is not None:
                x *= np.broadcast_to(f(np.arange(npg[b] * 128), S[b]), (npg[b] * 128,))[None, :, None]
            c, s = kv4.quantise(_val(_bits(x, dtype), dtype))
            rows.append(kv4.values(c, s)[:, :S[b]])
            pages[..., side * kv4.SIDE:(side + 1) * kv4.SIDE] = kv4.pack(c).reshape(Hkv, npg[b], kv4.SIDE)
            sc = pages[..., 2 * kv4.SIDE:].reshape(Hkv, npg[b], 128, 16)
            sc[..., 8 * side:8 * side + 8] = s.view(np.uint8).reshape(Hkv, npg[b], 128, 8)
            pages[..., 2 * kv4.SIDE:] = sc.reshape(Hkv, npg[b], 2048)
        blocks = ids[at:at + npg[b]]
        at += npg[b]
        table[b, :npg[b]] = torch.from_numpy(blocks)
        pool.raw()[torch.from_numpy(blocks.astype(np.int64)).cuda(), 0] = torch.from_numpy(pages.transpose(1, 0, 2)).cuda()
        k.append(rows[0])
        v.append(rows[1])
    x = rng.standard_normal((B, T, Hq, 128))
    if qf is not None:
        x *= np.broadcast_to(qf(np.arange(T)), (T,))[None, :, None, None]
    bits = _bits(x, dtype)
    x, gt = _val(bits, dtype), None
    if gains:
        f = kv4.norm_rows32(x)
        g = [_bits(rng.standard_normal(128) * 0.1 + 3, dtype) for _ in range(2)]
        for gb in g:
            f = f * (np.float32(1) + _val(gb, dtype).astype(np.float32))
        x, gt = _val(_bits(x.astype(np.float32) * f, dtype), dtype), tuple(_act(gb, dtype) for gb in g)
    o = torch.full((B, T, Hq * 128), 3.0, dtype=ctx.torch_dtype, device="cuda")
    attn.full_prefill(ctx, pool, table, 0, torch.tensor(pos0, dtype=torch.int32, device="cuda"), _act(bits, dtype).view(B, T, Hq * 128), o, gains=gt)
    ctx.check()
    got = _out(o, dtype).reshape(B, T, Hq, 128)
    want, bound = np.zeros_like(got), np.zeros_like(got)
    for b in range(B):
        seen = np.arange(S[b])[None] <= pos0[b] + np.arange(T)[:, None]
        for h in range(Hq):
            want[b, :, h], bound[b, :, h] = kv4.relu2(x[b, :, h], k[b][h // G], v[b][h // G], seen, kv4.U16[dtype], wround=4, dot=2.0 ** -11)
    return got, want, bound


SIZES = {
    "scores past fp16": dict(kf=lambda t, S: 30.0, qf=lambda t: 60.0),
    "scores of 1e8": dict(kf=lambda t, S: 3000.0, qf=lambda t: 3000.0),
    "one large query row": dict(kf=lambda t, S: 8.0, qf=lambda t: np.where(t == 100, 3000.0, 1.0)),
    "one large key in the chunk": dict(kf=lambda t, S: np.where(t == S - 30, 10000.0, 1.0), qf=lambda t: 8.0),
    "one large key ahead of it": dict(kf=lambda t, S: np.where(t == 3, 10000.0, 1.0), qf=lambda t: 8.0),
    "values near the type's largest": dict(vf=lambda t, S: 12000.0),
    "small queries beside large ones": dict(kf=lambda t, S: 100.0, qf=lambda t: np.where(t % 2, 1000.0, 1e-3)),
}
SIZES_BF16 = {
    "queries past fp16": dict(qf=lambda t: 1e8),
    "keys and values past fp16": dict(kf=lambda t, S: 1e5, vf=lambda t, S: 1e5),
    "one value past fp16 in the chunk": dict(vf=lambda t, S: np.where(t == S - 2, 1e5, 1.0)),
    "scores of 1e16": dict(kf=lambda t, S: 1e5, qf=lambda t: 1e11),
    "all of it": dict(kf=lambda t, S: 1e5, vf=lambda t, S: 1e5, qf=lambda t: 1e6),
}


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("what", list(SIZES) + list(SIZES_BF16))
@pytest.mark.parametrize("Hq,Hkv,pos0,T", [(2, 1, [300, 0], 333), (8, 2, [3000], 200), (4, 1, [9000], 40)])
def test_prefill_rows_of_every_size(dtype, what, Hq, Hkv, pos0, T):
    """Scores whose squares, and rows that fp16 does not hold, with whole chunks, and page ranges in clusters and through the scratch."""
    if dtype == "f16" and what in SIZES_BF16:
        return
    got, want, bound = _prefill_case(dtype, Hq, Hkv, pos0, T, 5, **{**SIZES, **SIZES_BF16}[what])
    keep = np.abs(want) < 65504.0 * (1 - 2.0 ** -9) if dtype == "f16" else np.ones(want.shape, bool)   # (what the output type holds)
    assert keep.mean() > 0.9
    _within(np.where(keep, got, 0), np.where(keep, want, 0), bound, what)
    # as a whole: 2^-11 for each of key, value, weight and output (the weight's key twice), at most doubled, and bf16's own half step
    some = np.abs(want).max(-1) > 0                        # (a token at position 0 whose only score is negative has zeros)
    rms = np.sqrt((np.where(keep, got - want, 0)[some] ** 2).sum(-1) / (np.where(keep, want, 0)[some] ** 2).sum(-1))
    assert np.median(rms) < (2.0 ** -10 if dtype == "f16" else 2.0 ** -8.5), np.median(rms)


@pytest.mark.parametrize("Hq,Hkv,pos0,T", [(8, 2, [6000], 1024), (2, 1, [12000], 700)])
def test_prefill_large_rows_shared_among_ctas(Hq, Hkv, pos0, T):
    """Large keys in some page ranges of a unit and none in others, and gains that make large queries."""
    got, want, bound = _prefill_case("bf16", Hq, Hkv, pos0, T, 6, kf=lambda t, S: np.where(t % 1500 == 77, 3000.0, 1.0),
                                     vf=lambda t, S: np.where(t == S - 1000, 1e5, 1.0), gains=True)
    _within(got, want, bound, "rows")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,pos0,T", [(2, 1, [300, 0], 333), (8, 2, [3000], 200)])
def test_prefill_small_rows(dtype, Hq, Hkv, pos0, T):
    """Scores of about 0.01, all of them: the weights, of 1e-4, keep their leading bits."""
    got, want, bound = _prefill_case(dtype, Hq, Hkv, pos0, T, 5, kf=lambda t, S: 1e-2)
    # beside the other roundings a weight is off by half of fp16's smallest step, 2^-25 x 2^3, times a value of 6 or less and the keys seen
    seen = np.stack([p + 1 + np.arange(T) for p in pos0])[:, :, None, None]
    _within(got, want, bound + seen * 6 * 2.0 ** -22 / np.sqrt(128.0), "small rows")
    # as a whole, for the tokens that see many: 2^-22 of 1e-4 at random is 2^-9.5 at most, halved by the rounding's distribution
    late = np.arange(T) > T // 2
    rms = np.sqrt(((got - want)[:, late] ** 2).mean() / (want[:, late] ** 2).mean())
    assert rms < (2.0 ** -9 if dtype == "f16" else 2.0 ** -8), rms


@pytest.mark.parametrize("gains", [False, True])
def test_prefill_one_query_element_past_fp16(gains):
    """Every key has a negative element where a bf16 query is just too large for fp16: minus infinity there, which weighs nothing, and a positive score
    in earnest for half of them."""
    import torch
    from embla_metal_b200 import attn
    rng = np.random.default_rng(2)
    n, T = 300, 40
    ctx, pool = attn.Attention(2, 1, attn.BF16, 1, 384), attn.KVPool(1, 1, 3, attn.KV_INT4)
    rows = rng.standard_normal((2, 1, n, 128))
    rows[0, ..., 0] = -2.0
    kb = _bits(rows, "bf16")
    t = _act(kb, "bf16")
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    ctx.kv_append(pool, table, 0, torch.zeros(1, dtype=torch.int32, device="cuda"), t[0], t[1], norm_k=False)
    k, v = (kv4.values(*kv4.quantise(_val(kb[i, 0], "bf16"))) for i in range(2))
    assert (k[:, 0] < 0).all()
    x = np.sign(rng.standard_normal((T, 2, 128))) * 1.0e6
    x[..., 0] = 2.2e6
    gt = None
    if gains:                                              # raw queries of size 1 whose gains make those
        g = [_bits(np.full(128, 1.0e3 - 1), "bf16"), _bits(np.full(128, 1.1e3 - 1), "bf16")]
        x = np.sign(x) * np.where(np.arange(128) == 0, 1.0, 0.5)
        gt = tuple(_act(gb, "bf16") for gb in g)
    qb = _bits(x, "bf16")
    q = _val(qb, "bf16")
    if gains:
        f = kv4.norm_rows32(q)
        for gb in g:
            f = f * (np.float32(1) + _val(gb, "bf16").astype(np.float32))
        q = _val(_bits(q.astype(np.float32) * f, "bf16"), "bf16")
    assert (q[..., 0] > 2.1e6).all() and (np.abs(q[..., 1:]) < 2.09e6).all()
    o = torch.zeros(1, T, 256, dtype=torch.bfloat16, device="cuda")
    attn.full_prefill(ctx, pool, table, 0, torch.tensor([n - T], dtype=torch.int32, device="cuda"), _act(qb, "bf16").view(1, T, 256), o, gains=gt)
    ctx.check()
    got = _out(o, "bf16").reshape(T, 2, 128)
    seen = np.arange(n)[None] <= n - T + np.arange(T)[:, None]
    for h in range(2):
        want, bound = kv4.relu2(q[:, h], k, v, seen, kv4.U16["bf16"], wround=4, dot=2.0 ** -11)
        _within(got[:, h], want, bound, f"head {h}")


# ---- value groups of different sizes, in the decodes -------------------------------------------------------------
def _group_pages(rng, pool, table, b, lens, Hkv, layer, vf):
    """Pages of sequence b: keys ~ N(0, 1), values ~ N(0, 1) x vf [4] by group; returns their values."""
    import torch
    npg = (lens[b] + 127) // 128
    pages = np.zeros((Hkv, npg, kv4.PAGE), np.uint8)
    out = []
    for side, f in ((0, np.ones(4)), (1, np.asarray(vf, float))):
        x = (rng.standard_normal((Hkv, npg * 128, 4, 32)) * f[:, None]).astype(np.float16).astype(np.float64).reshape(Hkv, npg * 128, 128)
        c, s = kv4.quantise(x)
        out.append(kv4.values(c, s)[:, :lens[b]])
        pages[..., side * kv4.SIDE:(side + 1) * kv4.SIDE] = kv4.pack(c).reshape(Hkv, npg, kv4.SIDE)
        sc = pages[..., 2 * kv4.SIDE:].reshape(Hkv, npg, 128, 16)
        sc[..., 8 * side:8 * side + 8] = s.view(np.uint8).reshape(Hkv, npg, 128, 8)
        pages[..., 2 * kv4.SIDE:] = sc.reshape(Hkv, npg, 2048)
    pool.raw()[table[b, :npg].long(), layer] = torch.from_numpy(pages.transpose(1, 0, 2)).cuda()
    return out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("vf", [[100.0, 1e-3, 1.0, 1e-2], [12000.0, 1e-3, 1e-3, 1e-2], [5.0, 1e-3, 15.0, 1e-2]])
@pytest.mark.parametrize("Hq,Hkv,lens", [(8, 2, [1000, 37]), (16, 2, [9000] * 3 + [300] * 8)])
def test_decodes_keep_small_groups_beside_large_ones(dtype, vf, Hq, Hkv, lens):
    """A group of values far above the others changes nothing for them: full decode (as a cluster and in runs, with key scores and without) and
    sparse decode."""
    import torch
    from embla_metal_b200 import attn
    rng = np.random.default_rng(len(lens))
    B, G, width = len(lens), Hq // Hkv, (max(lens) + 127) // 128
    ctx = attn.Attention(Hq, Hkv, DT[dtype], B, width * 128)
    pool = attn.KVPool(1, Hkv, B * width, attn.KV_INT4)
    table = torch.from_numpy(rng.permutation(B * width).reshape(B, width).astype(np.int32)).cuda()
    kv = [_group_pages(rng, pool, table, b, lens, Hkv, 0, vf) for b in range(B)]
    qt, qv, _ = _queries(rng, B, Hq, dtype, 0)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    o = torch.zeros(B, Hq * 128, dtype=ctx.torch_dtype, device="cuda")
    sc = torch.zeros(B, Hkv, width * 128, device="cuda")
    idx = np.zeros((B, Hkv, 1152), np.int32)
    for b in range(B):
        if lens[b] > 1152:
            for h in range(Hkv):
                idx[b, h, :1024] = np.sort(rng.permutation(lens[b] - 128)[:1024])
            idx[b, :, 1024:] = np.arange(lens[b] - 128, lens[b])

    def check(what, form):
        ctx.check()
        got = _out(o, dtype).reshape(B, Hq, 128)
        rms = []
        for b in range(B):
            for h in range(Hkv):
                k, v = (x[h] for x in kv[b])
                if form == "sparse" and lens[b] > 1152:
                    k, v = k[idx[b, h]], v[idx[b, h]]
                qb = qv[b, h * G:(h + 1) * G]
                if form == "sparse":
                    want, bound = kv4.softmax(qb, k, v, kv4.U16[dtype])
                else:
                    want, bound = kv4.relu2(qb, k, v, np.ones((G, len(k)), bool), kv4.U16[dtype])
                _within(got[b, h * G:(h + 1) * G], want, bound, f"{what}, sequence {b}, kv head {h}")
                d = (got[b, h * G:(h + 1) * G] - want).reshape(G, 4, 32)
                rms.append(np.sqrt((d ** 2).sum((0, 2)) / (want.reshape(G, 4, 32) ** 2).sum((0, 2))))
        # each group as a whole: a weight's and an output's rounding (2^-11 each; bf16 2^-8; fp16 outputs of 1e-4 are subnormal: 2^-25)
        worst = np.max(rms, 0)
        limit = np.array([2.0 ** -10 if f > 5e-3 else 2.0 ** -8 for f in vf]) if dtype == "f16" else 2.0 ** -8
        assert (worst < limit).all(), (what, worst)

    ctx.full_decode(pool, table, ln, 0, qt, o)
    check("full decode", "full")
    ctx.full_decode(pool, table, ln, 0, qt, o, scores=sc)
    check("full decode with scores", "full")
    ctx.sparse_decode(pool, table, ln, 0, qt, o, idx=torch.from_numpy(idx).cuda())
    check("sparse decode", "sparse")


# ---- pages that are not there ------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("lens,page", [([400], 1), ([400], 3), ([9000] * 6 + [300] * 9, 2), ([9000] * 6 + [300] * 9, 70)])
def test_scores_of_a_bad_block_are_zeros(bad, lens, page):
    """The call is reported, and leaves no score of an earlier one behind: those of the positions in the bad block are 0, all others right."""
    import torch
    from embla_metal_b200 import attn
    rng, ctx, pool, table, k, v = _setup("bf16", 8, 2, lens, 19)
    qt, qv, _ = _queries(rng, len(lens), 8, "bf16", 0)
    table[0, page] = bad
    o = torch.zeros(len(lens), 1024, dtype=torch.bfloat16, device="cuda")
    sc = torch.full((len(lens), 2, table.shape[1] * 128 + 5), -7.0, device="cuda")
    ctx.full_decode(pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1, qt, o, scores=sc)
    with pytest.raises(attn.EmblaError) as e:
        ctx.check()
    assert e.value.status == attn.BAD_ARG
    for b, n in enumerate(lens):
        for h in range(2):
            row = sc[b, h].cpu().numpy().astype(np.float64)
            qb = qv[b, 4 * h:4 * h + 4]
            want, err = (qb @ k[b][h].T).max(0), kv4.DOT * (np.abs(qb) @ np.abs(k[b][h]).T).max(0)
            if b == 0:
                want[128 * page:128 * page + 128] = err[128 * page:128 * page + 128] = 0.0
            assert (row[n:] == -7.0).all()
            _within(row[:n], want, err, f"scores of sequence {b}, kv head {h}")


# ---- queries of any size -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("size", [1e4, 1e7, 1e8, 1e10, 1e25, 1e33, 1e37])
def test_sparse_decode_of_large_queries(size):
    """Softmax over scores that far apart: the value of the largest."""
    import torch
    lens = [900, 64]
    rng, ctx, pool, table, k, v = _setup("bf16", 4, 2, lens, 3)
    q, qv, _ = _queries(rng, 2, 4, "bf16", 0, factor=size)
    o = torch.zeros(2, 512, dtype=torch.bfloat16, device="cuda")
    ctx.sparse_decode(pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1, q, o)
    ctx.check()
    got = _out(o, "bf16").reshape(2, 4, 128)
    for b in range(2):
        for h in range(4):
            best = np.argmax(k[b][h // 2] @ qv[b, h])
            want = v[b][h // 2][best]
            # the weight and its product with the scale in fp16, the sum of weights, the output
            _within(got[b, h], want, np.abs(want) * (3 * 2.0 ** -11 + 2.0 ** -8), f"sequence {b}, head {h}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["even", "one 2^8", "one 2^16", "wide", "sparse"])
def test_scores_of_uneven_rows(dtype, kind):
    """Key scores where one query element is far above the rest, where they span 2^24, and for keys of one code a group: off by at most 2^-16 of
    max |q| x sum |k|. A group's products are fp32 sums of 32 terms and a start value, of either sign and up to 15 max |q| s in size, where the
    pipe may truncate: 34 steps of 2^-24 of a partial sum that is 15 sqrt(32) max |q| s at most as a rule, at random 2^-15.1 max |q| s, and sum
    |k| of the group is 7 s or more: 2^-17.9. A query element is off by 2^-25 max |q|."""
    import torch
    from embla_metal_b200 import attn
    n = 4096
    for seed in range(2):
        rng = np.random.default_rng(seed)
        ctx = attn.Attention(2, 2, DT[dtype], 1, n)
        pool = attn.KVPool(1, 2, n // 128, attn.KV_INT4)
        pages = kv4.make_pages(rng, (n // 128, 1, 2))
        if kind == "sparse":
            codes = np.zeros((n // 128, 1, 2, 128, 4, 32), np.int8)
            np.put_along_axis(codes, rng.integers(0, 32, codes.shape[:-1])[..., None], 7, -1)
            pages[..., :8192] = kv4.pack(codes.reshape(*codes.shape[:-2], 128)).reshape(n // 128, 1, 2, 8192)
        pool.raw().copy_(torch.from_numpy(pages))
        x = rng.standard_normal((1, 2, 128))
        if kind in ("wide", "sparse"):
            x *= np.exp2(rng.uniform(-24, 0, x.shape))
        if kind.startswith("one"):
            x *= 2.0 ** -3
            x[:, :, 5] *= 2.0 ** float(kind[6:])
        bits = _bits(x, dtype)
        q = _val(bits, dtype)[0]
        o = torch.zeros(1, 256, dtype=ctx.torch_dtype, device="cuda")
        sc = torch.zeros(1, 2, n, device="cuda")
        ctx.full_decode(pool, torch.arange(n // 128, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda"), 0,
                        _act(bits, dtype).view(1, -1), o, scores=sc)
        ctx.check()
        k = kv4.page_values(pages[:, 0].transpose(1, 0, 2))[0].reshape(2, n, 128)
        bound = 2.0 ** -16 * np.abs(q).max(-1)[:, None] * np.abs(k).sum(-1)
        _within(sc[0].cpu().numpy().astype(np.float64), np.einsum("hd,hnd->hn", q, k), bound + 1e-30, kind)


@pytest.mark.parametrize("scores", [False, True])
@pytest.mark.parametrize("size", [1e4, 1e10, 1e15])
@pytest.mark.parametrize("lens", [[900, 64], [9000] * 5])
def test_full_decode_of_large_queries(size, lens, scores):
    """Weights up to 1e31: the same bounds as for small ones."""
    import torch
    rng, ctx, pool, table, k, v = _setup("bf16", 4, 2, lens, 3)
    B = len(lens)
    q, qv, _ = _queries(rng, B, 4, "bf16", 0, factor=size)
    o = torch.zeros(B, 512, dtype=torch.bfloat16, device="cuda")
    sc = torch.zeros(B, 2, table.shape[1] * 128, device="cuda") if scores else None
    ctx.full_decode(pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1, q, o, scores=sc)
    ctx.check()
    got = _out(o, "bf16").reshape(B, 2, 2, 128)
    for b in range(B):
        for h in range(2):
            qb = qv[b].reshape(2, 2, 128)[h]
            want, bound = kv4.relu2(qb, k[b][h], v[b][h], np.ones((2, lens[b]), bool), kv4.U16["bf16"])
            _within(got[b, h], want, bound, f"sequence {b}, kv head {h}")
            if scores:
                _within(sc[b, h, :lens[b]].cpu().numpy().astype(np.float64), (qb @ k[b][h].T).max(0), kv4.DOT * (np.abs(qb) @ np.abs(k[b][h]).T).max(0),
                        f"scores of sequence {b}, kv head {h}")
