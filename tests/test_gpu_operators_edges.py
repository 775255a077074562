"""The decoding operators on the GPU at the edges of their definitions, results written over buffers that hold other values
before. Tolerances as in test_gpu_operators.py."""
import numpy as np
import pytest
import torch  # noqa: F401  (before the plugin: both then use one HIP runtime)

from oracle import operators as oo
from oracle import stablehlo as sh
from ryft_amd import pjrt
from tests import operator_programs as op
from tests.test_gpu_operators import attention_error, close, device_buffers, span, sync

pytestmark = pytest.mark.gpu


def run_over(client, module, ins, outs):
    """The results of one execution into buffers that hold 7s before; outs: (shape, dtype)."""
    exe = client.compile(pjrt.Program.mlir(module))
    bufs = device_buffers(client, ins)
    res = device_buffers(client, [op.host(np.full(shape, 7.0), dt) for shape, dt in outs])
    exe.execute_into([span(b) for b in bufs], [span(b) for b in res])
    sync()
    return [sh.from_raw(b.to_numpy().view(np.uint16) if dt == "f16" else b.to_numpy(), dt).reshape(shape)
            for b, (shape, dt) in zip(res, outs)]


# ------------------------------------------------------------------------------------------------ more queries than keys
MORE_QUERIES = {
    "none": dict(new=[200], lengths=[0], heads=(4, 2)),
    "ten": dict(new=[200], lengths=[10], heads=(4, 2)),
    "behind": dict(new=[100, 3, 300, 0, 90], lengths=[150, 3, 0, 9, 20], heads=(4, 2)),
    "window": dict(new=[200, 70], lengths=[10, 100], heads=(4, 1), window=5),
    "capped": dict(new=[200, 70], lengths=[10, 100], heads=(5, 1), softcap=5.0, slopes=True),
    "not_causal": dict(new=[200, 70], lengths=[10, 0], heads=(4, 2), causal=False),
    # tiles alone fill the chip; ranges of keys; more sequences than a wavefront holds
    "many_tiles": dict(new=[20] * 8 + [300], lengths=[20] * 8 + [0], heads=(64, 64)),
    "ranges": dict(new=[200, 40], lengths=[10, 700], heads=(4, 2)),
    "many": dict(new=[30] * 66 + [200], lengths=[5] * 66 + [0], heads=(8, 8)),
}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", MORE_QUERIES)
def test_more_queries_than_keys(gpu_client, name, d, dtype):
    c = dict(MORE_QUERIES[name])
    new, lengths, heads = (c.pop(k) for k in ("new", "lengths", "heads"))
    module, ins = op.attention_case(new, lengths, *heads, d, 16, dtype, seed=len(name) + d, **c)
    (got,) = run_over(gpu_client, module, ins, [(ins[0].dims, dtype)])
    x = op.values(ins)
    want, = oo.paged_attention(x, op.config_of(module))
    close(got, want, dtype, attention_error(x, dtype), name)
    unseen = ~want.any(axis=(1, 2))
    assert unseen.any() and not got[unseen].any()                     # rows that see nothing are exactly zero
