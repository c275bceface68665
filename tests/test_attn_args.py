"""The packed calls of the Python binding without a GPU: an argument that is missing is the library's error, as in the calls that are not packed."""
import pytest
import torch

from embla_metal_b200 import attn


def test_missing_positions_are_the_library_s_error(monkeypatch):
    monkeypatch.setattr(attn, "_raw_stream", lambda: 0)
    ctx = attn.Attention.__new__(attn.Attention)
    ctx.handle, ctx._prefill_reserved = None, True
    pool = attn.KVPool.__new__(attn.KVPool)
    pool.handle = None
    x = torch.zeros(1, 1, 128, dtype=torch.float16)
    table = torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: ctx.kv_append(pool, table, 0, None, x, x), lambda: attn.full_prefill(ctx, pool, table, 0, None, x, x)):
        with pytest.raises(attn.EmblaError) as e:
            call()
        assert e.value.status == attn.BAD_ARG
