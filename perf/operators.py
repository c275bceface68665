"""The operators of the 4-bit KV cache and the copies of cache blocks, as cases to measure.

Definitions (both forms below and the CUDA kernels follow them)

* A 4-bit page holds 128 positions of one (layer, kv head), 18,432 bytes: K codes [128][64 B] | V codes [128][64 B] |
  scales float16 [128][8] (K groups 0-3, V groups 0-3). A row's 128 dims are four groups of 32 with a scale each. The
  32-bit word w of a row's codes holds dims 8w .. 8w+7 as two's complement nibbles; nibble n is dim 8w + (0,2,4,6,1,3,5,7)[n].
* Quantisation of a row x (rounded to the activation type; keys first RMS-normed where asked): per group
  s = float16(min(max|x| / 7, 65504)), code = clamp(rint(x / s), -7, 7), 0 where s is 0. Value: code * s.
* Full layers: w_j = max(q.k_j / sqrt(128), 0)^2 over the keys j a query sees, o = sum w_j v_j / (sqrt(128) + sum w_j).
  Key scores: max over the kv head's query heads of q.k_j. Sparse layers: softmax(q.k_j / sqrt(128)) over every key of a
  sequence of at most 1152, else over 1152 selected positions a kv head. A sequence without keys gives zeros.
* Queries may come raw: RMS norm over the head with gains (1 + g1)(1 + g2), rounded to the activation type.
"""
import math

import torch

own = False

HD, BLOCK, TOPK, RECENT = 128, 128, 1024, 128
CODES, PAGE = 8192, 18432
EPS = 1.1920929e-07
_DT = {"bf16": torch.bfloat16, "f16": torch.float16}
_NIBBLE_DIM = (0, 2, 4, 6, 1, 3, 5, 7)


# ---- cases ------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoded token of every sequence of a batch of 64, keys normed, into the cache, and read back: latency
        dict(name="append_read_64x1_bf16", op="append", dtype="bf16", hq=16, hkv=4, batch=64, tokens=1, base=4095, norm=True),
        # the prompt chunks of eight sequences, each starting inside a block
        dict(name="append_read_8x2048_f16", op="append", dtype="f16", hq=16, hkv=4, batch=8, tokens=2048, base=1000, norm=False),
        # one short sequence: latency of a decode launch
        dict(name="decode_1x1000_f16", op="decode", dtype="f16", hq=16, hkv=4, batch=1, ctx=1000, ragged=False, gains=False,
             scores=False),
        # 16 sequences of uneven lengths, an odd group of three query heads a kv head
        dict(name="decode_16x9001_g3_bf16", op="decode", dtype="bf16", hq=24, hkv=8, batch=16, ctx=9001, ragged=True, gains=False,
             scores=False),
        # the model's own shape (2 kv heads of 8 query heads, raw queries with both gains) that also scores the keys for
        # the sparse layers behind it
        dict(name="decode_8x32768_scores_bf16", op="decode", dtype="bf16", hq=16, hkv=2, batch=8, ctx=32768, ragged=False, gains=True,
             scores=True),
        # batched decode at full context
        dict(name="decode_64x32768_f16", op="decode", dtype="f16", hq=16, hkv=4, batch=64, ctx=32768, ragged=False, gains=False,
             scores=False),
        # a few sequences past the selection's length
        dict(name="sparse_4x9000_bf16", op="sparse", dtype="bf16", hq=16, hkv=2, batch=4, ctx=9000, ragged=True, gains=True),
        # the sparse layers of batched decode at full context
        dict(name="sparse_64x32768_f16", op="sparse", dtype="f16", hq=16, hkv=4, batch=64, ctx=32768, ragged=False, gains=False),
        # short uneven prompts of three sequences behind what they have cached
        dict(name="prefill_3x333_f16", op="prefill", dtype="f16", hq=16, hkv=4, batch=3, tokens=333, base=700, gains=False),
        # a whole prompt chunk at the end of a full context
        dict(name="prefill_1x2048_at30720_bf16", op="prefill", dtype="bf16", hq=16, hkv=4, batch=1, tokens=2048, base=30720,
             gains=False),
        # 48 sequences forked: each gets its own copy of the rows in its last block
        dict(name="copy_48_tails", op="copy", layers=6, hkv=4, copies=48, rows="ragged"),
        # blocks moved together so that the end of the pool comes free
        dict(name="copy_512_blocks", op="copy", layers=6, hkv=4, copies=512, rows="full"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "sparse", "prefill", "copy"])
    if op == "copy":
        return dict(op=op, layers=rng.randint(1, 6), hkv=rng.choice([1, 2, 4]), copies=_log(rng, 1, 512),
                    rows=rng.choice(["ragged", "full"]))
    hkv = rng.choice([1, 2, 4])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    if hkv * group > 16:
        group = 16 // hkv
    c = dict(op=op, dtype=rng.choice(["bf16", "f16"]), hq=hkv * group, hkv=hkv)
    if op == "append":
        tokens = _log(rng, 1, 2048)
        c.update(batch=_log(rng, 1, max(1, min(64, 16384 // tokens))), tokens=tokens, base=_log(rng, 1, 20000), norm=rng.random() < 0.5)
    elif op == "decode":
        scores = rng.random() < 0.3
        c.update(batch=_log(rng, 1, 16 if scores else 64), ctx=_log(rng, 1, 32768), ragged=rng.random() < 0.5, gains=rng.random() < 0.5,
                 scores=scores)
    elif op == "sparse":
        c.update(batch=_log(rng, 1, 64), ctx=_log(rng, 1, 32768), ragged=rng.random() < 0.5, gains=rng.random() < 0.5)
    else:
        tokens = _log(rng, 1, 2048)
        c.update(batch=_log(rng, 1, max(1, min(4, 2048 // tokens))), tokens=tokens, base=_log(rng, 1, 30720), gains=rng.random() < 0.5)
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------
def _quantise(x):
    """x float32 [..., 128], already rounded to the activation type -> codes int8 [..., 128], scales float16 [..., 4]."""
    g = x.unflatten(-1, (4, 32))
    top = g.abs().amax(-1)
    s = torch.where(torch.isfinite(top), (top / 7.0).clamp(max=65504.0), torch.nan).to(torch.float16)
    sf = s.float().unsqueeze(-1)
    c = torch.where(sf > 0, g / sf, torch.zeros_like(g)).round().clamp(-7, 7)
    return c.flatten(-2).to(torch.int8), s


def _pack(codes):
    """int8 codes [..., 128] -> uint8 [..., 64]."""
    n = (codes.to(torch.int32) & 15).unflatten(-1, (16, 8))[..., list(_NIBBLE_DIM)].unflatten(-1, (4, 2))
    return (n[..., 0] | (n[..., 1] << 4)).to(torch.uint8).flatten(-2)


def _fill_pages(flat, gen, dev):
    """Random 4-bit pages: rows of keys and values ~ N(0, 1), one key in a hundred four times as large."""
    step = 4096
    for i in range(0, flat.shape[0], step):
        part = flat[i:i + step]
        n = part.shape[0]
        x = torch.randn(n, 2, BLOCK, HD, device=dev, generator=gen, dtype=torch.float16)
        big = torch.rand(n, BLOCK, 1, device=dev, generator=gen) < 0.01
        x[:, 0] *= torch.where(big, 4.0, 1.0).to(x.dtype)
        codes, s = _quantise(x.float())
        part[:, :2 * CODES] = _pack(codes).reshape(n, 2 * CODES)
        part[:, 2 * CODES:] = s.permute(0, 2, 1, 3).contiguous().view(torch.uint8).reshape(n, PAGE - 2 * CODES)


def _lens(case, gen, dev):
    """Keys a sequence has: all of them `ctx`, or uneven (the first the longest; with three or more, one without any)."""
    B, ctx = case["batch"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * B
    u = torch.rand(B, generator=gen, device=dev).tolist()
    lens = [max(1, int(round(ctx * x))) for x in u]
    lens[0] = ctx
    if B >= 3:
        lens[-1] = 0
    return lens


def _inputs(case, seed, pages):
    """The case's inputs; `pages(layers, hkv, blocks)` gives the zeroed bytes [blocks][layers][hkv][page] of a pool."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, hkv = case["op"], case["hkv"]
    st = dict(case=case)
    if op == "copy":
        n = case["copies"]
        blocks = 2 * n + 3
        st["raw"] = pages(case["layers"], hkv, blocks)
        st["raw"].copy_(torch.randint(0, 256, st["raw"].shape, device=dev, dtype=torch.uint8, generator=gen))
        ids = torch.randperm(blocks, generator=gen, device=dev).to(torch.int32)
        st["src"], st["dst"] = ids[:n].contiguous(), ids[n:2 * n].contiguous()
        st["rows"] = torch.randint(1, BLOCK, (n,), device=dev, dtype=torch.int32, generator=gen) if case["rows"] == "ragged" else None
        return st
    dt, B, hq = _DT[case["dtype"]], case["batch"], case["hq"]
    st["dtype"] = dt
    if op in ("append", "prefill"):
        T = case["tokens"]
        p0 = [case["base"]] + [max(0, case["base"] - 37 * b - 11) for b in range(1, B)]
        st["pos0_host"] = p0
        st["pos0"] = torch.tensor(p0, dtype=torch.int32, device=dev)
        st["max_len"] = max(p0) + T
        npg = [(p + T + BLOCK - 1) // BLOCK for p in p0]
    else:
        lens = _lens(case, gen, dev)
        st["lens_host"] = lens
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        st["max_len"] = case["ctx"]
        npg = [(n + BLOCK - 1) // BLOCK for n in lens]
    width = max(npg)
    ids = torch.randperm(sum(npg) + 1, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32, device=dev)
    at = 0
    for b in range(B):
        table[b, :npg[b]] = ids[at:at + npg[b]]
        at += npg[b]
    st["table"] = table
    st["raw"] = pages(1, hkv, sum(npg) + 1)
    if op == "append":
        qkv = torch.randn(B, T, (hq + 2 * hkv) * HD, device=dev, generator=gen).to(dt)   # the projections' rows: q, k, v
        st["k"], st["v"] = qkv[..., hq * HD:(hq + hkv) * HD], qkv[..., (hq + hkv) * HD:]
        st["k_out"] = torch.zeros(B, T, hkv * HD, dtype=dt, device=dev)
        st["v_out"] = torch.zeros_like(st["k_out"])
        return st
    _fill_pages(st["raw"].view(-1, PAGE), gen, dev)
    shape = (B, case["tokens"], hq * HD) if op == "prefill" else (B, hq * HD)
    st["q"] = torch.randn(shape, device=dev, generator=gen).to(dt)
    st["gains"] = tuple((torch.randn(HD, device=dev, generator=gen) * 0.05).to(dt) for _ in range(2)) if case["gains"] else None
    st["o"] = torch.zeros_like(st["q"])
    if op == "decode" and case["scores"]:
        st["scores"] = torch.zeros(B, hkv, width * BLOCK, device=dev)
    if op == "sparse":
        idx = torch.zeros(B, hkv, TOPK + RECENT, dtype=torch.int32, device=dev)
        for b in range(B):
            n = lens[b]
            if n > TOPK + RECENT:
                for h in range(hkv):
                    idx[b, h, :TOPK] = torch.randperm(n - RECENT, generator=gen, device=dev)[:TOPK].sort().values
                idx[b, :, TOPK:] = torch.arange(n - RECENT, n, device=dev)
        st["idx"] = idx
    return st


def prepare(case, seed):
    if not own:
        return _inputs(case, seed, lambda layers, hkv, blocks: torch.zeros(blocks, layers, hkv, PAGE, dtype=torch.uint8, device="cuda"))
    from embla_metal_b200 import attn
    box = {}

    def pages(layers, hkv, blocks):
        box["pool"] = attn.KVPool(layers, hkv, blocks, attn.KV_INT4, attn.SCALE_F16)
        return box["pool"].raw()

    st = _inputs(case, seed, pages)
    st["pool"] = box["pool"]
    if case["op"] == "copy":
        st["ctx"] = attn.Attention(case["hkv"], case["hkv"], attn.F16, 1, BLOCK)
    else:
        st["ctx"] = attn.Attention(case["hq"], case["hkv"], attn.BF16 if case["dtype"] == "bf16" else attn.F16, case["batch"],
                                   max(1, st["max_len"]))
    return st


# ---- the framework's operators ----------------------------------------------------------------------------------
def _run_own(st):
    from embla_metal_b200 import attn
    case, ctx, pool = st["case"], st["ctx"], st["pool"]
    op = case["op"]
    if op == "copy":
        ctx.copy_blocks(pool, st["src"], st["dst"], st["rows"])
        return st["raw"]
    if op == "append":
        ctx.kv_append(pool, st["table"], 0, st["pos0"], st["k"], st["v"], norm_k=case["norm"])
        ctx.kv_read(pool, st["table"], 0, st["pos0"], st["k_out"], st["v_out"])
        return st["k_out"], st["v_out"]
    if op == "decode":
        ctx.full_decode(pool, st["table"], st["lens"], 0, st["q"], st["o"], gains=st["gains"], scores=st.get("scores"),
                        max_seq_len=st["max_len"])
        return (st["o"], st["scores"]) if case["scores"] else st["o"]
    if op == "sparse":
        ctx.sparse_decode(pool, st["table"], st["lens"], 0, st["q"], st["o"], idx=st["idx"], gains=st["gains"], max_seq_len=st["max_len"])
        return st["o"]
    attn.full_prefill(ctx, pool, st["table"], 0, st["pos0"], st["q"], st["o"], gains=st["gains"])
    return st["o"]


# ---- the plain form ---------------------------------------------------------------------------------------------
def _norm_rows(x):
    """RMS norm factors [..., 1] of float32 rows [..., 128]: partial sums of dims l, l + 32, l + 64, l + 96, then l = 0 .. 31."""
    sq = (x * x).unflatten(-1, (4, 32))
    part = ((sq[..., 0, :] + sq[..., 1, :]) + sq[..., 2, :]) + sq[..., 3, :]
    tot = part[..., 0]
    for lane in range(1, 32):
        tot = tot + part[..., lane]
    return (1.0 / (tot / float(HD) + EPS).sqrt()).unsqueeze(-1)


def _unpack(codes, scales):
    """uint8 [..., 64], float16 [..., 4] -> float32 values [..., 128]."""
    lo, hi = codes & 15, codes >> 4
    n = torch.stack([lo, hi], -1).flatten(-2).unflatten(-1, (16, 8)).to(torch.int8)
    n = (n ^ 8) - 8
    order = [_NIBBLE_DIM.index(d) for d in range(8)]
    c = n[..., order].flatten(-2)
    return (c.float().unflatten(-1, (4, 32)) * scales.float().unsqueeze(-1)).flatten(-2)


def _rows(raw, table_row, n, first=0):
    """Keys and values float32 [hkv, n, 128] of positions first .. first + n - 1."""
    b0, b1 = first // BLOCK, (first + n + BLOCK - 1) // BLOCK
    pages = raw[table_row[b0:b1].long(), 0]                                   # [blocks, hkv, page]
    hkv = pages.shape[1]
    s = pages[..., 2 * CODES:].contiguous().view(torch.float16).unflatten(-1, (BLOCK, 8))
    out = []
    for side in range(2):
        c = pages[..., side * CODES:(side + 1) * CODES].unflatten(-1, (BLOCK, 64))
        x = _unpack(c, s[..., 4 * side:4 * side + 4]).transpose(0, 1).reshape(hkv, -1, HD)
        out.append(x[:, first - b0 * BLOCK:first - b0 * BLOCK + n])
    return out


def _queries(st):
    q = st["q"].float().unflatten(-1, (-1, HD))
    if st["gains"] is None:
        return q
    g = _norm_rows(q)
    for gain in st["gains"]:
        g = g * (1.0 + gain.float())
    return (q * g).to(st["dtype"]).float()


def _run_plain(st):
    case, raw = st["case"], st["raw"]
    op = case["op"]
    root = math.sqrt(HD)
    if op == "copy":
        hkv, L = case["hkv"], case["layers"]
        if st["rows"] is None:
            raw[st["dst"].long()] = raw[st["src"].long()]
            return raw
        keep = torch.arange(BLOCK, device=raw.device) < st["rows"].unsqueeze(1)              # [n, 128]
        new, old = raw[st["src"].long()], raw[st["dst"].long()]
        code = keep[:, None, None, None, :, None]
        a = torch.where(code, new[..., :2 * CODES].unflatten(-1, (2, BLOCK, 64)), old[..., :2 * CODES].unflatten(-1, (2, BLOCK, 64)))
        b = torch.where(keep[:, None, None, :, None], new[..., 2 * CODES:].unflatten(-1, (BLOCK, 16)),
                        old[..., 2 * CODES:].unflatten(-1, (BLOCK, 16)))
        n = st["src"].shape[0]
        raw[st["dst"].long()] = torch.cat([a.reshape(n, L, hkv, 2 * CODES), b.reshape(n, L, hkv, PAGE - 2 * CODES)], -1)
        return raw
    hq, hkv, B = case["hq"], case["hkv"], case["batch"]
    G = hq // hkv
    if op == "append":
        T = case["tokens"]
        outs = []
        codes, scales = [], []
        for x, norm in ((st["k"], case["norm"]), (st["v"], False)):
            x = x.float().unflatten(-1, (hkv, HD))                                            # [B, T, hkv, 128]
            if norm:
                x = (x * _norm_rows(x)).to(st["dtype"]).float()
            c, s = _quantise(x)
            codes.append(_pack(c))
            scales.append(s)
            outs.append((c.float().unflatten(-1, (4, 32)) * s.float().unsqueeze(-1)).flatten(-2).to(st["dtype"]).reshape(B, T, hkv * HD))
        pos = st["pos0"].long().unsqueeze(1) + torch.arange(T, device=raw.device)             # [B, T]
        block = st["table"].long().gather(1, pos // BLOCK).unsqueeze(-1)
        row = (pos % BLOCK).unsqueeze(-1)
        head = torch.arange(hkv, device=raw.device)
        for side in range(2):
            raw[..., side * CODES:(side + 1) * CODES].unflatten(-1, (BLOCK, 64))[:, 0][block, head, row] = codes[side]
        sc = torch.cat(scales, -1).view(torch.uint8)                                          # [B, T, hkv, 16]
        raw[..., 2 * CODES:].unflatten(-1, (BLOCK, 16))[:, 0][block, head, row] = sc
        return tuple(outs)
    q = _queries(st)
    if op == "prefill":
        T = case["tokens"]
        o = torch.empty_like(st["q"])
        for b in range(B):
            p0 = st["pos0_host"][b]
            k, v = _rows(raw, st["table"][b], p0 + T)
            seen = torch.arange(p0 + T, device=raw.device) <= (p0 + torch.arange(T, device=raw.device)).unsqueeze(1)
            for h in range(hq):
                w = (q[b, :, h] @ k[h // G].t() / root).clamp(min=0.0).square() * seen
                o[b, :, h * HD:(h + 1) * HD] = ((w @ v[h // G]) / (root + w.sum(-1, keepdim=True))).to(o.dtype)
        return o
    o = torch.zeros_like(st["q"])
    scores = torch.zeros_like(st["scores"]) if op == "decode" and case["scores"] else None
    for b in range(B):
        n = st["lens_host"][b]
        if n == 0:
            continue
        qb = q[b].view(hkv, G, HD)
        k, v = _rows(raw, st["table"][b], n)
        if op == "sparse":
            if n > TOPK + RECENT:
                at = st["idx"][b].long().unsqueeze(-1).expand(-1, -1, HD)
                k, v = k.gather(1, at), v.gather(1, at)
            s = qb @ k.transpose(1, 2) / root
            w = (s - s.amax(-1, keepdim=True)).exp()
            r = (w @ v) / w.sum(-1, keepdim=True)
        else:
            s = qb @ k.transpose(1, 2)
            if scores is not None:
                scores[b, :, :n] = s.amax(1)
            w = (s / root).clamp(min=0.0).square()
            r = (w @ v) / (root + w.sum(-1, keepdim=True))
        o[b] = r.reshape(-1).to(o.dtype)
    return (o, scores) if scores is not None else o


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits ----------------------------------------------------------------------------------
def _page_values(pages):
    """pages uint8 [n, PAGE] -> float64 keys and values [n, 128, 128], word by word."""
    n = pages.shape[0]
    words = pages[:, :2 * CODES].contiguous().view(torch.int32).view(n, 2, BLOCK, 16)
    scales = pages[:, 2 * CODES:].contiguous().view(torch.float16).view(n, BLOCK, 2, 4).double()
    out = torch.empty(n, 2, BLOCK, 16, 8, dtype=torch.float64, device=pages.device)
    for nib, dim in enumerate(_NIBBLE_DIM):
        x = (words >> (4 * nib)) & 15
        out[..., dim] = torch.where(x >= 8, x - 16, x).double()
    out = out.view(n, 2, BLOCK, 4, 32) * scales.transpose(1, 2).unsqueeze(-1)
    out = out.view(n, 2, BLOCK, HD)
    return out[:, 0], out[:, 1]


def _unit(x):
    return x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()


def exact(case, seed):
    st = _inputs(case, seed, lambda layers, hkv, blocks: torch.zeros(blocks, layers, hkv, PAGE, dtype=torch.uint8, device="cuda"))
    op, hkv = case["op"], case["hkv"]
    if op == "copy":
        raw = st["raw"]
        src, dst = st["src"].tolist(), st["dst"].tolist()
        rows = [BLOCK] * len(src) if st["rows"] is None else st["rows"].tolist()
        out = raw.clone()
        for a, b, r in zip(src, dst, rows):
            for lo, width in ((0, 64), (CODES, 64), (2 * CODES, 16)):
                out[b, :, :, lo:lo + width * r] = raw[a, :, :, lo:lo + width * r]
        return out
    hq, B, dt = case["hq"], case["batch"], st["dtype"]
    G, root = hq // hkv, math.sqrt(HD)
    if op == "append":
        res = []
        for x, norm in ((st["k"], case["norm"]), (st["v"], False)):
            x = x.double().reshape(B, case["tokens"], hkv, HD)
            if norm:
                x = _unit(x).to(dt).double()
            x = x.view(B, case["tokens"], hkv, 4, 32)
            s = (x.abs().amax(-1, keepdim=True) / 7).clamp(max=65504.0).to(torch.float16).double()
            c = torch.where(s > 0, torch.round(x / torch.where(s > 0, s, 1.0)), 0.0).clamp(-7, 7)
            res.append((c * s).reshape(B, case["tokens"], hkv * HD))
        return tuple(res)
    q = st["q"].double().unflatten(-1, (hq, HD))
    if st["gains"] is not None:
        q = (_unit(q) * (1 + st["gains"][0].double()) * (1 + st["gains"][1].double())).to(dt).double()
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=q.device)
    scores = torch.zeros(st["scores"].shape, dtype=torch.float64, device=q.device) if "scores" in st else None
    for b in range(B):
        n = st["pos0_host"][b] + case["tokens"] if op == "prefill" else st["lens_host"][b]
        for h in range(hkv if n else 0):
            k, v = _page_values(st["raw"][st["table"][b, :(n + BLOCK - 1) // BLOCK].long(), 0, h])
            k, v = k.reshape(-1, HD)[:n], v.reshape(-1, HD)[:n]
            heads = range(h * G, (h + 1) * G)
            if op == "prefill":
                last = st["pos0"][b] + torch.arange(case["tokens"], device=q.device)
                hidden = torch.arange(n, device=q.device)[None, :] > last[:, None]
                for i in heads:
                    w = torch.relu(torch.einsum("td,jd->tj", q[b, :, i], k) / root) ** 2
                    w = w.masked_fill(hidden, 0.0)
                    out[b, :, i * HD:(i + 1) * HD] = torch.einsum("tj,jd->td", w, v) / (root + w.sum(1))[:, None]
                continue
            if op == "sparse" and n > TOPK + RECENT:
                at = st["idx"][b, h].long()
                k, v = k[at], v[at]
            s = torch.einsum("gd,jd->gj", q[b, h * G:(h + 1) * G], k)
            if scores is not None:
                scores[b, h, :n] = s.max(0).values
            if op == "sparse":
                r = torch.softmax(s / root, 1) @ v
            else:
                w = torch.relu(s / root) ** 2
                r = (w @ v) / (root + w.sum(1))[:, None]
            out[b, h * G * HD:(h + 1) * G * HD] = r.reshape(-1)
    return (out, scores) if scores is not None else out


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    op, hkv = case["op"], case["hkv"]
    if op == "copy":
        rows = BLOCK / 2 if case["rows"] == "ragged" else BLOCK
        return {"bytes": 2 * case["copies"] * case["layers"] * hkv * rows * (PAGE / BLOCK), "flops": 0}
    row = PAGE // BLOCK                                                     # bytes of a key and its value: 144
    hq, B = case["hq"], case["batch"]
    if op == "append":
        n = B * case["tokens"] * hkv
        return {"bytes": n * (4 * HD + row + 4 * HD), "flops": n * 2 * HD * 4}
    if op == "prefill":
        T, p0 = case["tokens"], [case["base"]] + [max(0, case["base"] - 37 * b - 11) for b in range(1, B)]
        seen = sum(T * p + T * (T + 1) // 2 for p in p0)
        return {"bytes": sum(p + T for p in p0) * hkv * row + 4 * B * T * hq * HD, "flops": 4 * HD * hq * seen}
    keys = B * case["ctx"] * (0.5 if case["ragged"] else 1.0)
    if op == "sparse":
        keys = min(keys, B * (TOPK + RECENT))
        return {"bytes": keys * hkv * (row + 4) + 4 * B * hq * HD, "flops": 4 * HD * hq * keys}
    return {"bytes": keys * hkv * (row + (4 if case["scores"] else 0)) + 4 * B * hq * HD, "flops": 4 * HD * hq * keys}
