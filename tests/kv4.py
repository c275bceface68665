"""Plain restatement of the 4-bit cache in numpy, 64 bits: the page format, the quantisation, and the attentions over it with a
bound on what the kernels' roundings may move each output by."""
import numpy as np

GROUP, PAGE, SIDE = 32, 18432, 8192
NIBBLE_DIM = (0, 2, 4, 6, 1, 3, 5, 7)
U16 = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}     # half a step of the storage type, relative


def quantise(x):
    """x [..., 128] (values of a 16-bit type) -> codes int8 [..., 128], scales float16 [..., 4]."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], 4, GROUP)
    top = np.abs(g).max(-1)                                        # (numpy's max keeps a NaN)
    with np.errstate(invalid="ignore", over="ignore"):
        s = np.where(np.isfinite(top), np.minimum(top / 7, 65504.0), np.nan).astype(np.float16)
    sf = s.astype(np.float64)[..., None]
    with np.errstate(invalid="ignore", divide="ignore"):
        c = np.where(sf > 0, np.rint(g / np.where(sf > 0, sf, 1.0)), 0.0)
    return np.clip(np.nan_to_num(c), -7, 7).astype(np.int8).reshape(x.shape), s


def pack(codes):
    """int8 [..., 128] -> uint8 [..., 64]."""
    c = (codes.astype(np.uint8) & 15).reshape(*codes.shape[:-1], 16, 8)[..., list(NIBBLE_DIM)]
    return (c[..., 0::2] | (c[..., 1::2] << 4)).reshape(*codes.shape[:-1], 64)


def unpack(rows):
    """uint8 [..., 64] -> int8 [..., 128]."""
    n = np.stack([rows & 15, rows >> 4], -1).reshape(*rows.shape[:-1], 16, 8)
    out = np.empty(n.shape, np.int8)
    out[..., list(NIBBLE_DIM)] = ((n ^ 8).astype(np.int8) - 8)
    return out.reshape(*rows.shape[:-1], 128)


def split_pages(pages):
    """uint8 [..., PAGE] -> k codes, v codes int8 [..., 128, 128], k scales, v scales float16 [..., 128, 4]."""
    lead = pages.shape[:-1]
    kc = unpack(pages[..., :SIDE].reshape(*lead, 128, 64))
    vc = unpack(pages[..., SIDE:2 * SIDE].reshape(*lead, 128, 64))
    sc = np.ascontiguousarray(pages[..., 2 * SIDE:]).view(np.float16).reshape(*lead, 128, 8)
    return kc, vc, sc[..., :4], sc[..., 4:]


def values(codes, scales):
    with np.errstate(invalid="ignore"):              # (a group that holds no numbers has a NaN scale)
        return codes.astype(np.float64) * np.repeat(scales.astype(np.float64), GROUP, -1)


def page_values(pages):
    kc, vc, ks, vs = split_pages(pages)
    return values(kc, ks), values(vc, vs)


def make_pages(rng, shape, kscale=1.0, vscale=1.0):
    """Random pages uint8 [*shape, PAGE] of rows ~ N(0, 1) times the factors, rounded to float16."""
    out = np.zeros((*shape, PAGE), np.uint8)
    for side, f in ((0, kscale), (1, vscale)):
        x = (rng.standard_normal((*shape, 128, 128)) * f).astype(np.float16)
        c, s = quantise(x)
        out[..., side * SIDE:(side + 1) * SIDE] = pack(c).reshape(*shape, SIDE)
        sc = out[..., 2 * SIDE:].reshape(*shape, 128, 16)
        sc[..., 8 * side:8 * side + 8] = s.view(np.uint8).reshape(*shape, 128, 8)
        out[..., 2 * SIDE:] = sc.reshape(*shape, 2048)
    return out


def norm_rows32(x):
    """RMS norm factors in float32, in the kernels' order: dims l + 32 i by i, then the lanes l."""
    x = np.asarray(x, np.float32)
    sq = (x * x).reshape(*x.shape[:-1], 4, 32)
    part = ((sq[..., 0, :] + sq[..., 1, :]) + sq[..., 2, :]) + sq[..., 3, :]
    tot = part[..., 0]
    for i in range(1, 32):
        tot = tot + part[..., i]
    return (np.float32(1) / np.sqrt(tot / np.float32(128) + np.float32(1.1920929e-07), dtype=np.float32))[..., None]


# ---- attentions. q [n, 128], k, v [S, 128] float64, seen bool [n, S]. The kernels' roundings, to first order:
#  * a dot is a fp32 sum of 128 products of fp16 values (queries scaled by a power of two) with four group scales: off by at most
#    dot = DOT x sum |q k|, DOT = 2^-17 (128 steps and the offset of the codes, 72 / 7 of the products' size, of 2^-24 each,
#    where the tensor pipe may truncate: twice that);
#  * `wround` roundings to fp16 of 2^-11 each between a weight and its product with a value (the weight itself, the
#    weight times the value's scale), fp32 sums of n terms: n 2^-24 of the sum of magnitudes;
#  * the quotient is rounded once to the output type.
DOT = 2.0 ** -17


def _finish(w, dw, v, sink, out_u, wround):
    den = w.sum(1, keepdims=True) + sink
    den = np.where(den == 0, 1.0, den)
    o = (w @ v) / den
    mag = (w @ np.abs(v)) / den
    rel = wround * 2.0 ** -11 + 2 * w.shape[1] * 2.0 ** -24
    err = (dw @ np.abs(v) + np.abs(o) * dw.sum(1, keepdims=True)) / den + mag * rel
    # (a subnormal output is off by at most its own step: fp16 2^-25)
    return o, 1.02 * (err + np.abs(o) * out_u + 2.0 ** -25)


def relu2(q, k, v, seen, out_u, wround=2, dot=DOT):
    """o = sum w v / (sqrt(128) + sum w), w = relu(q.k / sqrt(128))^2, and the bound."""
    s = (q @ k.T) / np.sqrt(128.0)
    ds = dot * (np.abs(q) @ np.abs(k).T) / np.sqrt(128.0)
    w = np.where(seen, np.maximum(s, 0.0) ** 2, 0.0)
    dw = np.where(seen, 2 * np.maximum(s + ds, 0.0) * ds + ds * ds, 0.0) * (s + ds > 0)
    # weights far below the largest of their row are kept to 2^-25 of it or better
    dw = dw + np.where(seen & (s > 0), 2.0 ** -21 * w.max(1, keepdims=True, initial=0.0), 0.0)
    return _finish(w, dw, v, np.sqrt(128.0), out_u, wround)


def softmax(q, k, v, out_u, wround=2, dot=DOT):
    """o = softmax(q.k / sqrt(128)) v and the bound; no keys: zeros."""
    if k.shape[0] == 0:
        return np.zeros((q.shape[0], 128)), np.zeros((q.shape[0], 128))
    s = (q @ k.T) / np.sqrt(128.0)
    ds = dot * (np.abs(q) @ np.abs(k).T) / np.sqrt(128.0)
    m = s.max(1, keepdims=True)
    w = np.exp(s - m)
    # exp2 of a fp32 argument: the argument's rounding times its size, and 2 ulp of the function
    dw = w * (np.expm1(2 * ds.max(1, keepdims=True)) + (np.abs(s - m) + 4) * 2.0 ** -22) + 2.0 ** -21
    return _finish(w, dw, v, 0.0, out_u, wround)
