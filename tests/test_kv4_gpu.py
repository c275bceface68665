"""The 4-bit cache (EMBLA_KV_INT4) and the copies of pool blocks on the GPU, against the 64-bit restatement in kv4.py."""
import ctypes as C

import numpy as np
import pytest

from oracle import oracle as orc
from tests import kv4, util

pytestmark = pytest.mark.gpu

DT = {"f16": orc.F16, "bf16": orc.BF16}


def _bits(x, dtype):
    return orc.to_bits(np.asarray(x, np.float32), DT[dtype])


def _val(bits, dtype):
    return orc.from_bits(bits, DT[dtype]).astype(np.float64)


def _act(bits, dtype):
    return util.act_tensor(bits, DT[dtype])


def _out(t, dtype):
    return _val(util.act_bits(t), dtype)


def _setup(dtype, Hq, Hkv, lens, seed, layers=2, max_batch=None, extra=3, vscale=1.0, kscale=1.0, width=None):
    """Context, pool, permuted table and the pages of sequences of `lens` keys in layer 1; everything behind the last key is noise with
    NaN scales."""
    import torch
    from embla_metal_b200 import attn
    rng = np.random.default_rng(seed)
    B = len(lens)
    npg = [(n + 127) // 128 for n in lens]
    width = width or max(1, max(npg))
    ctx = attn.Attention(Hq, Hkv, DT[dtype], max_batch or B, max(1, width * 128))
    pool = attn.KVPool(layers, Hkv, sum(npg) + extra, attn.KV_INT4, attn.SCALE_F16)
    raw = pool.raw()
    raw.copy_(torch.from_numpy(rng.integers(0, 256, tuple(raw.shape), dtype=np.uint8)))
    ids = rng.permutation(sum(npg) + extra).astype(np.int32)
    table = np.zeros((B, width), np.int32)
    k, v, at = [], [], 0
    for b in range(B):
        pages = kv4.make_pages(rng, (Hkv, npg[b]), kscale, vscale)
        tail = lens[b] % 128
        if tail:                                  # behind the last key: any codes, scales NaN and infinite
            sc = pages[:, -1, 2 * kv4.SIDE:].reshape(Hkv, 128, 16)
            sc[:, tail:] = np.array([0xff, 0x7f, 0x00, 0x7c] * 4, np.uint8)
            codes = pages[:, -1, :2 * kv4.SIDE].reshape(Hkv, 2, 128, 64)
            codes[:, :, tail:] = rng.integers(0, 256, (Hkv, 2, 128 - tail, 64), dtype=np.uint8)
            pages[:, -1] = np.concatenate([codes.reshape(Hkv, -1), sc.reshape(Hkv, -1)], -1)
        blocks = ids[at:at + npg[b]]
        at += npg[b]
        table[b, :npg[b]] = blocks
        if npg[b]:
            raw[torch.from_numpy(blocks.astype(np.int64)).cuda(), layers - 1] = torch.from_numpy(pages.transpose(1, 0, 2)).cuda()
        kv = kv4.page_values(pages)
        k.append(kv[0].reshape(Hkv, -1, 128)[:, :lens[b]])
        v.append(kv[1].reshape(Hkv, -1, 128)[:, :lens[b]])
    return rng, ctx, pool, torch.from_numpy(table).cuda(), k, v


def _queries(rng, B, Hq, dtype, gains, factor=1.0, pad=64):
    """q rows [B, Hq*128 + pad] (strided) on the device, their values after the norm, and the gains."""
    bits = _bits(rng.standard_normal((B, Hq * 128 + pad)) * factor, dtype)
    x = _val(bits[:, :Hq * 128], dtype).reshape(B, Hq, 128)
    if not gains:
        return _act(bits, dtype), x, None
    g = [_bits(rng.standard_normal(128) * 0.1, dtype) for _ in range(gains)]
    f = kv4.norm_rows32(x)
    for gb in g:
        f = f * (np.float32(1) + orc.from_bits(gb, DT[dtype]))
    xn = _val(_bits(x.astype(np.float32) * f, dtype), dtype)
    gt = (_act(g[0], dtype), _act(g[1], dtype) if gains == 2 else None)
    return _act(bits, dtype), xn, gt


def _within(got, want, bound, what):
    d = np.abs(got - want)
    assert np.isfinite(got).all(), f"{what}: not finite"
    worst = np.unravel_index(np.argmax(d - bound), d.shape)
    assert (d <= bound).all(), f"{what}: off by {d[worst]:.3e} at {worst}, bound {bound[worst]:.3e}, value {want[worst]:.3e}"


# ---- append and read ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_tokens,pos0,norm", [(1, [0, 127], True), (1, [128, 500], False), (3, [126, 5], True), (130, [1, 300], False),
                                                (257, [127, 0], True)])
def test_append_and_read(dtype, n_tokens, pos0, norm):
    import torch
    from embla_metal_b200 import attn
    rng = np.random.default_rng(n_tokens + norm)
    Hkv, B, width = 3, 2, 5
    ctx = attn.Attention(6, Hkv, DT[dtype], B, width * 128)
    pool = attn.KVPool(2, Hkv, B * width + 1, attn.KV_INT4, attn.SCALE_F16)
    raw = pool.raw()
    raw.copy_(torch.from_numpy(rng.integers(0, 256, tuple(raw.shape), dtype=np.uint8)))
    table = rng.permutation(B * width + 1)[:B * width].reshape(B, width).astype(np.int32)
    x = rng.standard_normal((2, B, n_tokens, Hkv, 128)) * np.exp(rng.uniform(-4, 4, (2, B, n_tokens, Hkv, 1)))
    x[0, 0, 0, 0] = 0.0                                  # a zero row
    x[1, 0, 0, 1, 32:64] = 0.0                           # a zero group
    x[1, 1, 0, 0] *= 1e-7                                # scales below the smallest normal, and to zero
    x[1, 1, 0, 1, 64:96] = 60000.0 if dtype == "f16" else 3e37   # scale saturates in bf16
    bits = _bits(x, dtype)
    rows = np.zeros((2, B, n_tokens, Hkv * 128 + 40), bits.dtype)
    rows[..., :Hkv * 128] = bits.reshape(2, B, n_tokens, -1)
    t = _act(rows, dtype)
    before = raw.cpu().numpy().copy()
    p0 = torch.tensor(pos0, dtype=torch.int32, device="cuda")
    ctx.kv_append(pool, torch.from_numpy(table).cuda(), 1, p0, t[0], t[1], norm_k=norm)
    ctx.check()
    want = before.copy()
    val = _val(bits, dtype)
    if norm:
        val[0] = _val(_bits(val[0].astype(np.float32) * kv4.norm_rows32(val[0]), dtype), dtype)
    codes, scales = kv4.quantise(val)
    packed = kv4.pack(codes)
    for b in range(B):
        for i in range(n_tokens):
            pos = pos0[b] + i
            pg = want[table[b, pos // 128], 1]
            r = pos % 128
            for side in range(2):
                pg[:, side * 8192 + r * 64:side * 8192 + r * 64 + 64] = packed[side, b, i]
                at = 16384 + r * 16 + side * 8
                pg[:, at:at + 8] = scales[side, b, i].view(np.uint8)
    assert np.array_equal(raw.cpu().numpy(), want)
    out = torch.full((2, B, n_tokens, Hkv * 128 + 8), 7.0, dtype=ctx.torch_dtype, device="cuda")
    ctx.kv_read(pool, torch.from_numpy(table).cuda(), 1, p0, out[0][..., :Hkv * 128], out[1][..., :Hkv * 128])
    ctx.check()
    got = util.act_bits(out)
    back = _bits(kv4.values(codes, scales), dtype).reshape(2, B, n_tokens, -1)
    neg0 = np.uint16(0x8000)                             # (-0 and 0 stand for the same value)
    assert np.array_equal(np.where(got[..., :Hkv * 128] == neg0, 0, got[..., :Hkv * 128]), np.where(back == neg0, 0, back))
    assert (_val(got[..., Hkv * 128:], dtype) == 7.0).all()


def test_append_marks_what_is_not_a_number():
    import torch
    from embla_metal_b200 import attn
    ctx = attn.Attention(1, 1, attn.BF16, 1, 128)
    pool = attn.KVPool(1, 1, 1, attn.KV_INT4)
    x = torch.ones(1, 3, 128, dtype=torch.bfloat16, device="cuda")
    x[0, 0, 5] = float("nan")
    x[0, 1, 40] = float("inf")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    p0 = torch.zeros(1, dtype=torch.int32, device="cuda")
    ctx.kv_append(pool, table, 0, p0, x, x, norm_k=False)
    k, v = torch.empty_like(x), torch.empty_like(x)
    ctx.kv_read(pool, table, 0, p0, k, v)
    ctx.check()
    for t in (k, v):
        nan = torch.isnan(t[0]).cpu().numpy()
        want = np.zeros((3, 128), bool)
        want[0, :32] = True
        want[1, 32:64] = True
        assert np.array_equal(nan, want)
        assert (t[0].cpu().float().numpy()[~want] == 1.0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["int8", "int8_f32", "16bit"])
def test_read_of_the_other_pools(dtype, kind):
    import torch
    from embla_metal_b200 import attn
    rng = np.random.default_rng(3)
    Hkv, B, T = 2, 2, 150
    ctx = attn.Attention(4, Hkv, DT[dtype], B, 512)
    pool = attn.KVPool(2, Hkv, 8, attn.KV_16BIT if kind == "16bit" else attn.KV_INT8, attn.SCALE_F32 if kind == "int8_f32" else attn.SCALE_F16)
    bits = _bits(rng.standard_normal((2, B, T, Hkv * 128)), dtype)
    t = _act(bits, dtype)
    table = torch.from_numpy(rng.permutation(8).reshape(2, 4).astype(np.int32)).cuda()
    p0 = torch.tensor([100, 3], dtype=torch.int32, device="cuda")
    ctx.kv_append(pool, table, 1, p0, t[0], t[1], norm_k=False)
    out = torch.zeros_like(t)
    ctx.kv_read(pool, table, 1, p0, out[0], out[1])
    ctx.check()
    if kind == "16bit":
        assert np.array_equal(util.act_bits(out), bits)
        return
    c, s = orc.quantize_rows(bits.reshape(-1, 128), DT[dtype], norm=False)
    if kind == "int8":
        s = s.astype(np.float16).astype(np.float32)
    want = _bits(c.astype(np.float32) * s[:, None], dtype).reshape(bits.shape)
    assert np.array_equal(_out(out, dtype), _val(want, dtype))


# ---- full layers, decode -----------------------------------------------------------------------------------------
def _check_full(ctx, pool, table, k, v, lens, rng, dtype, Hq, gains=0, scores=False, factor=1.0, q=None, max_len=0):
    import torch
    B, Hkv, G = len(lens), pool.n_kv_heads, Hq // pool.n_kv_heads
    qt, qv, gt = q or _queries(rng, B, Hq, dtype, gains, factor)
    o = torch.full((B, Hq * 128 + 24), 3.0, dtype=ctx.torch_dtype, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    sc = torch.full((B, Hkv, table.shape[1] * 128 + 5), -7.0, device="cuda") if scores else None
    ctx.full_decode(pool, table, ln, 1, qt, o, gains=gt, scores=sc, max_seq_len=max_len)
    ctx.check()
    got = _out(o, dtype)
    assert (got[:, Hq * 128:] == 3.0).all()
    got = got[:, :Hq * 128].reshape(B, Hq, 128)
    for b in range(B):
        for h in range(Hkv):
            qb = qv[b, h * G:(h + 1) * G]
            want, bound = kv4.relu2(qb, k[b][h], v[b][h], np.ones((G, lens[b]), bool), kv4.U16[dtype])
            _within(got[b, h * G:(h + 1) * G], want, bound, f"sequence {b} of {lens[b]} keys, kv head {h}")
            if scores:
                row = sc[b, h].cpu().numpy().astype(np.float64)
                assert (row[lens[b]:] == -7.0).all(), "scores behind the last key"
                if lens[b]:
                    want_s, err = (qb @ k[b][h].T).max(0), kv4.DOT * (np.abs(qb) @ np.abs(k[b][h]).T).max(0)
                    _within(row[:lens[b]], want_s, err + 1e-30, f"scores of sequence {b}, kv head {h}")
    return o, sc


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,lens", [
    (1, 1, [1]), (8, 1, [127]), (6, 2, [128, 1]), (4, 4, [129, 0, 2]), (16, 4, [1000]), (16, 2, [0]), (24, 8, [255, 4000, 16, 17, 640]),
    (10, 2, [9001]), (14, 2, [1152, 1153, 31, 33, 0, 385]), (16, 4, [300] * 40)])
def test_full_decode(dtype, Hq, Hkv, lens):
    rng, ctx, pool, table, k, v = _setup(dtype, Hq, Hkv, lens, Hq + len(lens))
    _check_full(ctx, pool, table, k, v, lens, rng, dtype, Hq)
    _check_full(ctx, pool, table, k, v, lens, rng, dtype, Hq, gains=2, scores=True, max_len=max(1, max(lens)))
    _check_full(ctx, pool, table, k, v, lens, rng, dtype, Hq, gains=1)


@pytest.mark.parametrize("scores", [False, True])
def test_full_decode_long(scores):
    lens = [32768, 20001]
    rng, ctx, pool, table, k, v = _setup("f16", 16, 2, lens, 8)
    _check_full(ctx, pool, table, k, v, lens, rng, "f16", 16, scores=scores)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kscale,vscale,qscale", [(1.0, 1.0, 60.0), (30.0, 1.0, 60.0), (1.0, 3000.0, 1.0), (1.0, 1e-3, 1.0), (30.0, 3000.0, 60.0),
                                                  (1e-2, 1e-3, 1e-2), (1.0, 3000.0, 1e-2)])
def test_full_decode_ranges(dtype, kscale, vscale, qscale):
    """Scores up to 10^5 and values up to 10^4 (weights up to 10^10: far outside fp16), and tiny ones."""
    lens = [700, 2500]
    rng, ctx, pool, table, k, v = _setup(dtype, 8, 2, lens, 5, kscale=kscale, vscale=vscale)
    q = _queries(rng, 2, 8, dtype, 0, qscale)
    _check_full(ctx, pool, table, k, v, lens, rng, dtype, 8, q=q, scores=True)


def test_full_decode_one_large_key_late():
    """A key near the end that outweighs all before it by 10^4: sums kept so far must give way exactly."""
    import torch
    lens = [1500]
    rng, ctx, pool, table, k, v = _setup("f16", 4, 1, lens, 6)
    q = _queries(rng, 1, 4, "f16", 0)
    raw = pool.raw()
    for pos in (20, 1300):
        pg = raw[int(table[0, pos // 128]), 1, 0]
        c, s = kv4.quantise((q[1][0, 1] * (10.0 if pos == 20 else 40.0)).astype(np.float16))
        r = pos % 128
        pg[r * 64:r * 64 + 64] = torch.from_numpy(kv4.pack(c)).cuda()
        pg[16384 + 16 * r:16384 + 16 * r + 8] = torch.from_numpy(s.view(np.uint8)).cuda()
        k[0][0, pos] = kv4.values(c, s)
    _check_full(ctx, pool, table, k, v, lens, rng, "f16", 4, q=q)


# ---- sparse layers, decode ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,lens,gains", [(16, 4, [1], 0), (16, 2, [127, 128, 129, 0], 2), (10, 2, [1151, 1152, 1153], 0), (8, 1, [5000], 1),
                                               (24, 8, [3000, 64, 1280, 0, 2], 2)])
def test_sparse_decode(dtype, Hq, Hkv, lens, gains):
    import torch
    rng, ctx, pool, table, k, v = _setup(dtype, Hq, Hkv, lens, 11 + Hq)
    _sparse(rng, ctx, pool, table, k, v, dtype, Hq, Hkv, lens, gains)


@pytest.mark.parametrize("kscale,vscale", [(30.0, 1.0), (1.0, 3000.0), (1.0, 1e-3)])
def test_sparse_decode_ranges(kscale, vscale):
    rng, ctx, pool, table, k, v = _setup("bf16", 8, 2, [1400, 300], 12, kscale=kscale, vscale=vscale)
    _sparse(rng, ctx, pool, table, k, v, "bf16", 8, 2, [1400, 300], 0)


def _sparse(rng, ctx, pool, table, k, v, dtype, Hq, Hkv, lens, gains):
    import torch
    B, G = len(lens), Hq // Hkv
    qt, qv, gt = _queries(rng, B, Hq, dtype, gains)
    idx = rng.integers(0, 2 ** 31, (B, Hkv, 1152))           # rows of short sequences are not read
    for b, n in enumerate(lens):
        if n > 1152:
            for h in range(Hkv):
                idx[b, h] = rng.permutation(n)[:1152]
    it = torch.from_numpy(idx.astype(np.int32)).cuda()
    o = torch.full((B, Hq * 128 + 8), 3.0, dtype=ctx.torch_dtype, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ctx.sparse_decode(pool, table, ln, 1, qt, o, idx=it, gains=gt)
    ctx.check()
    got = _out(o, dtype)
    assert (got[:, Hq * 128:] == 3.0).all()
    got = got[:, :Hq * 128].reshape(B, Hq, 128)
    for b, n in enumerate(lens):
        for h in range(Hkv):
            at = idx[b, h] if n > 1152 else np.arange(n)
            want, bound = kv4.softmax(qv[b, h * G:(h + 1) * G], k[b][h][at], v[b][h][at], kv4.U16[dtype])
            _within(got[b, h * G:(h + 1) * G], want, bound, f"sequence {b} of {n} keys, kv head {h}")


def test_sparse_decode_leaves_out_positions_outside_the_sequence():
    import torch
    from embla_metal_b200 import attn
    rng, ctx, pool, table, k, v = _setup("f16", 2, 1, [2000], 13)
    idx = np.arange(1152, dtype=np.int64)[None, None]
    idx[0, 0, 5], idx[0, 0, 700] = 2000, 2 ** 31 - 1
    qt, qv, _ = _queries(rng, 1, 2, "f16", 0)
    o = torch.zeros(1, 256, dtype=torch.float16, device="cuda")
    ctx.sparse_decode(pool, table, torch.tensor([2000], dtype=torch.int32, device="cuda"), 1, qt, o, idx=torch.from_numpy(idx.astype(np.int32)).cuda())
    with pytest.raises(attn.EmblaError) as e:
        ctx.check()
    assert e.value.status == attn.BAD_ARG
    at = np.delete(np.arange(1152), [5, 700])
    want, bound = kv4.softmax(qv[0], k[0][0][at], v[0][0][at], kv4.U16["f16"])
    _within(_out(o, "f16").reshape(2, 128), want, bound, "the other rows")
    ctx.check()


# ---- full layers, prefill ----------------------------------------------------------------------------------------
def _prefill(rng, ctx, pool, table, k, v, dtype, Hq, Hkv, pos0, T, gains, kscale=1.0):
    import torch
    from embla_metal_b200 import attn
    B, G = len(pos0), Hq // Hkv
    bits = _bits(rng.standard_normal((B, T, Hq * 128 + 16)), dtype)
    x = _val(bits[..., :Hq * 128], dtype).reshape(B, T, Hq, 128)
    gt = None
    if gains:
        g = [_bits(rng.standard_normal(128) * 0.1, dtype) for _ in range(2)]
        f = kv4.norm_rows32(x)
        for gb in g:
            f = f * (np.float32(1) + orc.from_bits(gb, DT[dtype]))
        x = _val(_bits(x.astype(np.float32) * f, dtype), dtype)
        gt = tuple(_act(gb, dtype) for gb in g)
    o = torch.full((B, T, Hq * 128 + 8), 3.0, dtype=ctx.torch_dtype, device="cuda")
    attn.full_prefill(ctx, pool, table, 1, torch.tensor(pos0, dtype=torch.int32, device="cuda"), _act(bits, dtype)[..., :Hq * 128], o, gains=gt)
    ctx.check()
    got = _out(o, dtype)
    assert (got[..., Hq * 128:] == 3.0).all()
    for b in range(B):
        S = pos0[b] + T
        seen = np.arange(S)[None] <= pos0[b] + np.arange(T)[:, None]
        for h in range(Hq):
            # on the tensor cores keys and values enter as fp16(code x scale): 2^-11 on every product of a dot and on every
            # value; a weight is rounded as relu(s) in fp16 (twice in its square), and squared in fp16: 4 in all
            want, bound = kv4.relu2(x[b, :, h], k[b][h // G], v[b][h // G], seen, kv4.U16[dtype], wround=4, dot=2.0 ** -11)
            _within(got[b, :, h * 128:(h + 1) * 128], want, bound, f"sequence {b} at {pos0[b]}, head {h}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,pos0,T,gains", [(1, 1, [0], 1, 0), (4, 2, [0, 130], 3, 1), (6, 2, [127], 129, 0), (8, 4, [300, 0, 77], 200, 1),
                                                 (2, 1, [1000], 256, 0), (16, 2, [5], 517, 0), (4, 4, [5000], 17, 1)])
def test_full_prefill(dtype, Hq, Hkv, pos0, T, gains):
    lens = [p + T for p in pos0]
    rng, ctx, pool, table, k, v = _setup(dtype, Hq, Hkv, lens, 17 + T)
    _prefill(rng, ctx, pool, table, k, v, dtype, Hq, Hkv, pos0, T, gains)


@pytest.mark.parametrize("Hq,Hkv,pos0,T", [(8, 2, [6000], 1024), (2, 1, [12000], 700)])
def test_full_prefill_shared_among_ctas(Hq, Hkv, pos0, T):
    lens = [p + T for p in pos0]
    rng, ctx, pool, table, k, v = _setup("bf16", Hq, Hkv, lens, 23)
    _prefill(rng, ctx, pool, table, k, v, "bf16", Hq, Hkv, pos0, T, 0)


# ---- copies of blocks --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["int4", "int8", "int8_f32", "16bit"])
@pytest.mark.parametrize("n,rows", [(1, None), (3, "ragged"), (9, None), (9, "ragged")])
def test_copy_blocks(kind, n, rows):
    import torch
    from embla_metal_b200 import attn
    rng = np.random.default_rng(n)
    kd = {"int4": attn.KV_INT4, "int8": attn.KV_INT8, "int8_f32": attn.KV_INT8, "16bit": attn.KV_16BIT}[kind]
    sb = 4 if kind == "int8_f32" else 2
    pool = attn.KVPool(3, 2, 2 * n + 2, kd, attn.SCALE_F32 if sb == 4 else attn.SCALE_F16)
    ctx = attn.Attention(2, 2, attn.F16, 1, 128)
    raw = pool.raw()
    raw.copy_(torch.from_numpy(rng.integers(0, 256, tuple(raw.shape), dtype=np.uint8)))
    ids = rng.permutation(2 * n + 2).astype(np.int32)
    src, dst = ids[:n], ids[n:2 * n]
    r = None
    if rows:
        r = rng.integers(1, 128, n).astype(np.int32)
        r[0], r[-1] = 1, 127
        if n > 4:
            r[1], r[2], r[3] = 0, 128, 500               # clamped to 128
    want = raw.cpu().numpy().copy()
    spans = {"int4": [(0, 64), (8192, 64), (16384, 16)], "16bit": [(0, 256), (32768, 256)]}.get(
        kind, [(0, 128), (16384, 128), (32768, sb), (32768 + 128 * sb, sb)])
    for i in range(n):
        m = 128 if r is None else min(128, int(r[i]))
        for at, w in spans:
            want[dst[i], :, :, at:at + w * m] = want[src[i], :, :, at:at + w * m]
    t = [torch.from_numpy(a).cuda() for a in (src, dst)]
    ctx.copy_blocks(pool, t[0], t[1], None if r is None else torch.from_numpy(r).cuda())
    ctx.check()
    assert np.array_equal(raw.cpu().numpy(), want)


def test_copy_blocks_leaves_out_bad_ids():
    import torch
    from embla_metal_b200 import attn
    pool = attn.KVPool(2, 1, 4, attn.KV_INT4)
    ctx = attn.Attention(1, 1, attn.F16, 1, 128)
    raw = pool.raw()
    raw.copy_(torch.arange(4, dtype=torch.uint8, device="cuda").view(4, 1, 1, 1).expand_as(raw))
    src = torch.tensor([0, -1, 1, 7], dtype=torch.int32, device="cuda")
    dst = torch.tensor([2, 3, 4, 3], dtype=torch.int32, device="cuda")
    ctx.copy_blocks(pool, src, dst)
    with pytest.raises(attn.EmblaError) as e:
        ctx.check()
    assert e.value.status == attn.BAD_ARG
    assert [int(raw[i].float().mean()) for i in range(4)] == [0, 1, 0, 3]
    ctx.copy_blocks(pool, src[:0], dst[:0])              # nothing to do
    ctx.check()


# ---- bad blocks, refusals ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [-1, 10 ** 6, 2 ** 31 - 1])
def test_bad_block_ids_are_reported_and_read_as_no_keys(bad):
    import torch
    from embla_metal_b200 import attn
    lens = [400]
    rng, ctx, pool, table, k, v = _setup("f16", 4, 2, lens, 19)
    table[0, 1] = bad
    raw = pool.raw()
    before = raw.clone()
    qt, qv, _ = _queries(rng, 1, 4, "f16", 0)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    p0 = torch.tensor([120], dtype=torch.int32, device="cuda")
    x = torch.ones(1, 20, 256, dtype=torch.float16, device="cuda")
    kk = [np.concatenate([a[:, :128], a[:, 256:]], 1) for a in (k[0], v[0])]

    def reported(fn):
        fn()
        with pytest.raises(attn.EmblaError) as e:
            ctx.check()
        assert e.value.status == attn.BAD_ARG
        ctx.check()

    o = torch.zeros(1, 512, dtype=torch.float16, device="cuda")
    reported(lambda: ctx.full_decode(pool, table, ln, 1, qt, o))
    for h in range(2):
        want, bound = kv4.relu2(qv[0, 2 * h:2 * h + 2], kk[0][h], kk[1][h], np.ones((2, 272), bool), kv4.U16["f16"])
        _within(_out(o, "f16").reshape(4, 128)[2 * h:2 * h + 2], want, bound, "full decode around a bad block")
    reported(lambda: ctx.sparse_decode(pool, table, ln, 1, qt, o))
    for h in range(2):
        want, bound = kv4.softmax(qv[0, 2 * h:2 * h + 2], kk[0][h], kk[1][h], kv4.U16["f16"])
        _within(_out(o, "f16").reshape(4, 128)[2 * h:2 * h + 2], want, bound, "sparse decode around a bad block")
    qp = qt[:, :512].reshape(1, 1, 512).contiguous()
    op = torch.zeros(1, 1, 512, dtype=torch.float16, device="cuda")
    reported(lambda: attn.full_prefill(ctx, pool, table, 1, torch.tensor([399], dtype=torch.int32, device="cuda"), qp, op))
    for h in range(2):
        want, bound = kv4.relu2(qv[0, 2 * h:2 * h + 2], kk[0][h], kk[1][h], np.ones((2, 272), bool), kv4.U16["f16"], wround=4, dot=2.0 ** -11)
        _within(_out(op, "f16").reshape(4, 128)[2 * h:2 * h + 2], want, bound, "prefill around a bad block")
    assert torch.equal(raw, before)
    reported(lambda: ctx.kv_append(pool, table, 1, p0, x, x, norm_k=False))
    after = raw.clone()
    page = int(table[0, 0])
    changed = (after != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [page]
    out = torch.full_like(x, 5.0)
    reported(lambda: ctx.kv_read(pool, table, 1, p0, out, torch.empty_like(out)))
    assert (out[0, :8] == 1.0).all() and (out[0, 8:] == 5.0).all()
    # positions behind the table's row
    reported(lambda: ctx.kv_append(pool, table, 1, torch.tensor([table.shape[1] * 128], dtype=torch.int32, device="cuda"), x, x))
    reported(lambda: ctx.kv_read(pool, table, 1, torch.tensor([-5], dtype=torch.int32, device="cuda"), out, torch.empty_like(out)))


def test_refusals():
    import torch
    from embla_metal_b200 import attn
    rng, ctx, pool, table, k, v = _setup("f16", 4, 2, [200], 20)
    ln = torch.tensor([200], dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 512, dtype=torch.float16, device="cuda")
    view = attn.Attention.view(table, ln, 1, 200)
    qd = attn.Attention.query(q)
    L = attn.lib()

    p = C.c_void_p(q.data_ptr())
    assert L.embla_attn_full_decode_noalloc(pool.handle, C.byref(view), C.byref(qd), 4, attn.F16, p, C.c_int64(512), None) == attn.UNSUPPORTED
    assert L.embla_attn_sparse_decode_int8(ctx.handle, pool.handle, C.byref(view), C.byref(qd), None, p, C.c_int64(512), None) == attn.UNSUPPORTED
    assert L.embla_attn_full_prefill_qk8(ctx.handle, pool.handle, C.byref(view), C.c_void_p(ln.data_ptr()), 1, C.byref(qd), C.c_int64(512), p,
                                         C.c_int64(512), C.c_int64(512), None) == attn.UNSUPPORTED
    pool8 = attn.KVPool(2, 2, 4, attn.KV_INT8)
    assert L.embla_attn_sparse_decode_int4(ctx.handle, pool8.handle, C.byref(view), C.byref(qd), None, p, C.c_int64(512), None) == attn.UNSUPPORTED
    far = attn.Attention.view(table, ln, 1, 5000)
    assert L.embla_attn_full_decode(ctx.handle, pool.handle, C.byref(far), C.byref(qd), p, C.c_int64(512), None, C.c_int64(0), None) == attn.BAD_ARG
    big = attn.Attention(4, 2, attn.F16, 1, 4096)
    assert L.embla_attn_sparse_decode_int4(big.handle, pool.handle, C.byref(attn.Attention.view(table, ln, 1, 2000)), C.byref(qd), None, p,
                                           C.c_int64(512), None) == attn.BAD_ARG        # past 1152 keys without the selected rows
    x = torch.zeros(1, 2, 256, dtype=torch.float16, device="cuda")
    p0 = torch.zeros(1, dtype=torch.int32, device="cuda")
    for args in [dict(token_stride=260, off=0), dict(token_stride=256, off=2)]:
        assert L.embla_kv_read(ctx.handle, pool.handle, C.byref(view), C.c_void_p(p0.data_ptr()), 1, C.c_void_p(x.data_ptr() + args["off"]),
                               C.c_void_p(x.data_ptr()), C.c_int64(args["token_stride"]), C.c_int64(512), None) == attn.BAD_ARG
    with pytest.raises(attn.EmblaError):
        ctx.kv_read(pool, table, 2, p0, x, x.clone())                                   # a layer the pool does not have
    with pytest.raises(ValueError):
        ctx.kv_read(pool, table, 1, p0, x.float(), x.float())
    for args in ((table, 1, p0, x.cpu(), x.cpu()), (table, 1, p0.cpu(), x, x.clone()), (table.long(), 1, p0, x, x.clone()), (table, 1, p0[:0], x, x.clone()),
                 (table, 1, p0, x.view(1, 1, 2, -1), x.view(1, 1, 2, -1))):
        with pytest.raises(ValueError):
            ctx.kv_read(pool, *args)
    with pytest.raises(ValueError):                                                     # rows too narrow for two kv heads
        ctx.kv_read(pool, table, 1, p0, x[..., :128], x[..., :128])
    shifted = torch.zeros(600, dtype=torch.float16, device="cuda")[1:513].view(1, 1, 512)
    with pytest.raises(attn.EmblaError) as e:                                           # queries that do not start on 16 bytes
        attn.full_prefill(ctx, pool, table, 1, p0, shifted, torch.zeros_like(shifted))
    assert e.value.status == attn.BAD_ARG
    with pytest.raises(ValueError):
        ctx.copy_blocks(pool, p0.long(), p0.long())
    with pytest.raises(ValueError):
        ctx.copy_blocks(pool, p0, torch.zeros(2, dtype=torch.int32, device="cuda"))
    w = attn.W4Weights(torch.zeros(512, 4, 4, dtype=torch.int32, device="cuda"), torch.zeros(512, 2, dtype=torch.bfloat16, device="cuda"),
                       torch.zeros(512, 2, dtype=torch.bfloat16, device="cuda"))
    wkv = attn.W4Weights(torch.zeros(256, 4, 4, dtype=torch.int32, device="cuda"), torch.zeros(256, 2, dtype=torch.bfloat16, device="cuda"),
                         torch.zeros(256, 2, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(attn.EmblaError) as e:
        ctx.qkv_project_full_step(w, wkv, wkv, torch.zeros(1, 128, dtype=torch.float16, device="cuda"),
                                  torch.zeros(1, 1024, dtype=torch.float16, device="cuda"), pool, table, ln, 1)
    assert e.value.status == attn.BAD_ARG                                               # (as for a 16-bit pool)


# ---- blocks taken out and put back, prompts shared, chunks scattered, batches ---------------------------------------
def test_exported_blocks_decode_the_same():
    import torch
    rng, ctx, pool, table, k, v = _setup("bf16", 8, 2, [700], 51, extra=8)
    q = _queries(rng, 1, 8, "bf16", 0)
    a, _ = _check_full(ctx, pool, table, k, v, [700], rng, "bf16", 8, q=q)
    free = [i for i in range(pool.num_blocks) if i not in table[0].tolist()][:6]
    host = [torch.empty(pool.block_bytes, dtype=torch.uint8).pin_memory() for _ in range(6)]
    for i in range(6):
        pool.export_block(int(table[0, i]), host[i])
    torch.cuda.synchronize()
    pool.raw()[table[0].long()] = 255
    for i, f in enumerate(free):
        pool.import_block(f, host[i])
    b, _ = _check_full(ctx, pool, torch.tensor([free], dtype=torch.int32, device="cuda"), k, v, [700], rng, "bf16", 8, q=q)
    assert torch.equal(a, b)


def test_prefix_store_keeps_blocks_of_a_4bit_pool():
    import torch
    from embla_metal_b200 import attn
    from embla_metal_b200.prefix import PrefixStore
    rng = np.random.default_rng(52)
    ctx = attn.Attention(4, 2, attn.F16, 2, 1024)
    pool = attn.KVPool(2, 2, 12, attn.KV_INT4)
    rings = [attn.Ring(2, 2, 1024, 128, torch.float16)]
    rings[0].k.normal_()
    rings[0].v.normal_()
    pool.raw().copy_(torch.from_numpy(rng.integers(0, 256, tuple(pool.raw().shape), dtype=np.uint8)))
    store = PrefixStore(1 << 28, pool, rings, n_kv_heads=2)
    tokens = list(range(500))
    store.save(0, [3, 1, 4, 5], tokens, 500, [500])
    before = pool.raw()[[3, 1, 4]].clone()
    start, _ = store.restore(1, [7, 8, 9, 10], tokens + [1, 2, 3])
    torch.cuda.synchronize()
    assert start == 384 and torch.equal(pool.raw()[[7, 8, 9]], before)


@pytest.mark.parametrize("T,p0,Hq,Hkv", [(64, 300, 8, 2), (300, 5000, 4, 1)])
def test_prefill_scattered_to_peers(T, p0, Hq, Hkv):
    import torch
    from embla_metal_b200 import attn
    rng, ctx, pool, table, k, v = _setup("bf16", Hq, Hkv, [p0 + T], 53)
    q = _act(_bits(rng.standard_normal((1, T, Hq * 128)), "bf16"), "bf16")
    pos0 = torch.tensor([p0], dtype=torch.int32, device="cuda")
    plain = torch.zeros_like(q)
    attn.full_prefill(ctx, pool, table, 1, pos0, q, plain)
    width = Hq * 128 + 256
    outs = [torch.full((T, width), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    attn.full_prefill_scatter(ctx, pool, table, 1, pos0, q, outs[0][:, 128:128 + Hq * 128].unsqueeze(0),
                              [o.data_ptr() + 256 for o in outs[1:]], width)
    ctx.check()
    for o in outs:
        assert torch.equal(o[:, 128:128 + Hq * 128], plain[0])
        assert (o[:, :128] == 7.0).all() and (o[:, 128 + Hq * 128:] == 7.0).all()


@pytest.mark.parametrize("batch,n", [(300, 40), (70, 700), (33, 129)])
def test_full_decode_of_many_sequences(batch, n):
    """More sequences than a warp has lanes, more units than SMs, lengths from 0 to n."""
    rng0 = np.random.default_rng(batch)
    lens = [int(x) for x in rng0.integers(0, n + 1, batch)]
    lens[0], lens[-1] = n, 0
    rng, ctx, pool, table, k, v = _setup("f16", 4, 2, lens, 54)
    _check_full(ctx, pool, table, k, v, lens, rng, "f16", 4, scores=True)


def test_all_sequences_empty():
    import torch
    from embla_metal_b200 import attn
    for batch, ctx_len in ((3, 128), (40, 8192)):
        ctx = attn.Attention(8, 2, attn.BF16, batch, ctx_len)
        pool = attn.KVPool(1, 2, 4, attn.KV_INT4)
        table = torch.zeros(batch, ctx_len // 128, dtype=torch.int32, device="cuda")
        ln = torch.zeros(batch, dtype=torch.int32, device="cuda")
        q = torch.randn(batch, 1024, device="cuda").bfloat16()
        for fn in (ctx.full_decode, ctx.sparse_decode):
            o = torch.full_like(q, 5.0)
            fn(pool, table, ln, 0, q, o, **({"idx": torch.zeros(batch, 2, 1152, dtype=torch.int32, device="cuda")} if fn == ctx.sparse_decode else {}))
            ctx.check()
            assert (o == 0).all()


def test_calls_repeat_bit_for_bit_and_in_a_graph():
    import torch
    lens = [5000, 300, 1200, 0, 77, 2048]
    rng, ctx, pool, table, k, v = _setup("bf16", 16, 4, lens, 55)
    q = _queries(rng, 6, 16, "bf16", 2)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    idx = torch.stack([torch.stack([torch.randperm(max(n, 1152), device="cuda")[:1152] for _ in range(4)]) for n in lens]).to(torch.int32)
    o, s = torch.zeros(6, 2048, dtype=torch.bfloat16, device="cuda"), torch.zeros(6, 2048, dtype=torch.bfloat16, device="cuda")
    sc = torch.zeros(6, 4, 5120, device="cuda")

    def calls():
        ctx.full_decode(pool, table, ln, 1, q[0], o, gains=q[2], scores=sc, max_seq_len=5000)
        ctx.sparse_decode(pool, table, ln, 1, q[0], s, idx=idx, gains=q[2], max_seq_len=5000)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
        side.synchronize()
        want = [t.clone() for t in (o, s, sc)]
        for _ in range(5):
            calls()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((o, s, sc), want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            calls()
        for t in (o, s, sc):
            t.zero_()
        for _ in range(3):
            graph.replay()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((o, s, sc), want))
        ctx.check()
    del graph


def test_append_of_rows_at_any_alignment():
    """Rows that do not start on 16 bytes, strides that are no multiple of 8 elements."""
    import torch
    from embla_metal_b200 import attn
    ctx = attn.Attention(2, 2, attn.F16, 2, 512)
    pools = [attn.KVPool(1, 2, 8, attn.KV_INT4) for _ in range(2)]
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    p0 = torch.tensor([3, 250], dtype=torch.int32, device="cuda")
    x = torch.randn(2, 2, 9, 256, device="cuda").half()
    odd = torch.zeros(2, 2, 9, 263, device="cuda", dtype=torch.float16)
    odd[..., 3:259] = x
    for norm in (False, True):
        ctx.kv_append(pools[0], table, 0, p0, x[0], x[1], norm_k=norm)
        ctx.kv_append(pools[1], table, 0, p0, odd[0][..., 3:259], odd[1][..., 3:259], norm_k=norm)
        ctx.check()
        assert torch.equal(pools[0].raw(), pools[1].raw())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("side", ["key", "value"])
def test_what_is_not_a_number_reaches_its_own_outputs_only(dtype, side):
    """A row with a NaN, appended at position 200 of the first of three sequences: the outputs of its kv head in that sequence are
    NaN, and a finite number everywhere else; one key and value that are infinite at a position nobody has reached change nothing."""
    import torch
    from embla_metal_b200 import attn
    Hq, Hkv, lens = 8, 2, [300, 300, 129]
    rng, ctx, pool, table, k, v = _setup(dtype, Hq, Hkv, lens, 41)
    tdt = torch.float16 if dtype == "f16" else torch.bfloat16
    row = torch.zeros(3, 1, Hkv * 128, dtype=tdt, device="cuda")
    row[0, 0, 128 + 70] = float("nan")
    row[1, 0, 5] = float("inf")
    ones = torch.ones_like(row)
    p0 = torch.tensor([200, 300, 129], dtype=torch.int32, device="cuda")
    ctx.kv_append(pool, table, 1, p0, row if side == "key" else ones, ones if side == "key" else row, norm_k=False)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.from_numpy(rng.standard_normal((3, Hq * 128)).astype(np.float32)).to("cuda", tdt)
    o = torch.zeros_like(q)

    def check(what):
        ctx.check()
        bad = torch.isnan(o.float()).view(3, Hkv, -1)
        assert not torch.isinf(o).any(), what
        assert not bad[1:].any() and not bad[0, 0].any(), what
        # (a value's NaN is in its group of 32 dims; a key's in every dim)
        own = torch.isnan(o.float()).view(3, Hq, 4, 32)[0, 4:, 70 // 32] if side == "value" else bad[0, 1]
        assert own.all(), what

    ctx.full_decode(pool, table, ln, 1, q, o)
    check("full decode")
    ctx.sparse_decode(pool, table, ln, 1, q, o)
    check("sparse decode")
    attn.full_prefill(ctx, pool, table, 1, ln - 1, q.view(3, 1, -1), o.view(3, 1, -1))
    check("prefill")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_tokens", [3, 5000])
def test_append_rounds_halves_to_even(dtype, n_tokens):
    """Rows whose quotients by their scale are whole numbers and halves, between -7 and 7, with scales down into fp16's subnormals."""
    import torch
    from embla_metal_b200 import attn
    rng = np.random.default_rng(n_tokens)
    npg = (n_tokens + 127) // 128
    ctx = attn.Attention(2, 2, DT[dtype], 1, npg * 128)
    pool = attn.KVPool(1, 2, npg, attn.KV_INT4, attn.SCALE_F16)
    # scales of 4 significant bits: times 13 / 2 or less they have 8, what bf16 holds
    s = rng.integers(8, 16, (2, n_tokens, 2, 4, 1)) * 2.0 ** rng.integers(-24, 9, (2, n_tokens, 2, 4, 1))
    m = rng.integers(-13, 14, (2, n_tokens, 2, 4, 32))
    m[..., 0] = np.where(rng.random(m[..., 0].shape) < 0.5, 14, -14)
    x = (np.take_along_axis(m, rng.permuted(np.broadcast_to(np.arange(32), m.shape), axis=-1), -1) * (s / 2)).reshape(2, 1, n_tokens, 2, 128)
    bits = _bits(x, dtype)
    keep = np.abs(_val(bits, dtype) - x) == 0            # (fp16: the smallest scales' halves are no numbers of the type)
    assert keep.mean() > 0.9
    t = _act(bits.reshape(2, 1, n_tokens, 256), dtype)
    table = torch.arange(npg, dtype=torch.int32, device="cuda").view(1, -1)
    ctx.kv_append(pool, table, 0, torch.zeros(1, dtype=torch.int32, device="cuda"), t[0], t[1], norm_k=False)
    ctx.check()
    codes, scales = kv4.quantise(_val(bits, dtype))
    assert (np.abs(x / np.repeat(s.reshape(2, 1, n_tokens, 2, 4), 32, -1)) % 1 == 0.5)[keep].mean() > 0.3
    raw = pool.raw()[:, 0].cpu().numpy()                 # [page][head][bytes]
    for side in range(2):
        got = raw[:, :, side * 8192:side * 8192 + 8192].reshape(npg, 2, 128, 64).transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:n_tokens]
        assert np.array_equal(got, kv4.pack(codes[side, 0]))
        sc = raw[:, :, 16384:].copy().view(np.float16).reshape(npg, 2, 128, 8).transpose(0, 2, 1, 3).reshape(-1, 2, 8)[:n_tokens]
        assert np.array_equal(sc[..., 4 * side:4 * side + 4], scales[side, 0])
