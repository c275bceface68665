"""The 4-bit cache without a GPU: the restatement the GPU tests compare with, and the refusals that come before any CUDA call."""
import ctypes as C

import numpy as np

from tests import kv4


def test_page_format_round_trip():
    rng = np.random.default_rng(0)
    codes = rng.integers(-7, 8, (5, 128)).astype(np.int8)
    assert np.array_equal(kv4.unpack(kv4.pack(codes)), codes)
    one = np.zeros((1, 128), np.int8)
    one[0, 10] = -3                                  # dim 10: word 1, its dim 2: nibble 1, the high half of byte 4
    row = kv4.pack(one)[0]
    assert row[4] == 0xd0 and row.sum() == 0xd0
    pages = kv4.make_pages(rng, (2, 3))
    kc, vc, ks, vs = kv4.split_pages(pages)
    assert kc.shape == (2, 3, 128, 128) and vs.shape == (2, 3, 128, 4)
    assert np.abs(kc).max() == 7 and np.abs(vc).max() == 7


def test_quantise_is_within_half_a_step():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((200, 128)) * np.exp(rng.uniform(-5, 5, (200, 1)))).astype(np.float16)
    c, s = kv4.quantise(x)
    err = np.abs(kv4.values(c, s) - x.astype(np.float64)).reshape(200, 4, 32)
    # half a step of the scale; the largest of a group loses at most the scale's own rounding on 7 steps as well
    assert (err <= s.astype(np.float64)[..., None] * (0.5 + 7 * 2.0 ** -11) + 2.0 ** -24).all()
    z, zs = kv4.quantise(np.zeros((1, 128), np.float16))
    assert not z.any() and not zs.any()


def test_refusals_without_a_gpu():
    from embla_metal_b200 import attn
    L = attn.lib()
    out = C.c_void_p()
    assert L.embla_kv_pool_create(1, 1, attn.KV_INT4, attn.SCALE_F32, 4, C.byref(out)) == attn.UNSUPPORTED
    assert b"fp16" in L.embla_last_error()
    assert L.embla_kv_pool_create(1, 1, 3, attn.SCALE_F16, 4, C.byref(out)) == attn.BAD_ARG
    assert L.embla_kv_read(None, None, None, None, 1, None, None, C.c_int64(0), C.c_int64(0), None) == attn.BAD_ARG
    assert L.embla_kv_copy_blocks(None, None, None, None, None, 1, None) == attn.BAD_ARG
    assert L.embla_attn_sparse_decode_int4(None, None, None, None, None, None, C.c_int64(0), None) == attn.BAD_ARG


def test_packed_records_are_the_header_s_structs():
    from embla_metal_b200 import attn
    assert attn._VIEW.size == C.sizeof(attn.KVView) and attn._QUERY.size == C.sizeof(attn.Query)
    v = attn.KVView.from_buffer_copy(attn._VIEW.pack(2 ** 40 + 1, 7, 2 ** 40 + 2, 3, 4, 5))
    assert [getattr(v, f[0]) for f in v._fields_] == [2 ** 40 + 1, 7, 2 ** 40 + 2, 3, 4, 5]
    q = attn.Query.from_buffer_copy(attn._QUERY.pack(2 ** 40 + 1, 2 ** 35, 1, 2, 2 ** 40 + 3, 0))
    assert [getattr(q, f[0]) for f in q._fields_] == [2 ** 40 + 1, 2 ** 35, 1, 2, 2 ** 40 + 3, None]
