"""The decoding operators without a GPU at the edges of their definitions."""
import numpy as np
import pytest

from ryft_amd import operators, pjrt


def attention(client, **kw):
    args = dict(tokens=3, sequences=2, q_heads=4, kv_heads=2, head_dim=64, pages=5, page_size=16, pages_per_sequence=4, scale=0.125)
    args.update(kw)
    return client.compile(pjrt.Program.mlir(operators.paged_attention_module(**args)))


# ------------------------------------------------------------------------------------------------ config
def test_every_finite_f32_is_a_scale_and_a_cap(compile_client):
    # the largest, as its shortest decimal form (which is larger than it is)
    most = float(np.finfo(np.float32).max)
    for kw in (dict(softcap=most), dict(scale=most), dict(scale=-most), dict(softcap=1e-45), dict(scale=1e-45)):
        attention(compile_client, **kw)
    for kw in (dict(softcap=np.inf), dict(scale=np.inf), dict(scale=-np.inf), dict(scale=np.nan)):
        with pytest.raises(pjrt.PjrtError) as e:
            attention(compile_client, **kw)
        assert e.value.code == pjrt.ErrorCode.INVALID_ARGUMENT and "out of range" in str(e.value)
