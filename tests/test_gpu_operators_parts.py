"""Paged attention over contexts that its kernels cut into parts: every unit of keys counts once. Values, bounds and what they
show are those of attention_parts.py; test_operators_parts.py holds that a lost or doubled unit is beyond the bound."""
import numpy as np
import pytest
import torch  # noqa: F401  (before the plugin: both then use one HIP runtime)

from ryft_amd import operators
from tests import attention_parts as ap
from tests import operator_programs as op
from tests.test_gpu_operators import run

pytestmark = pytest.mark.gpu


def within(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


@pytest.mark.parametrize("name, dtype", [(n, t) for n in ap.CASES for t in ("bf16", "f16")] + [("any", "f32"), ("step_one_head", "f32")])
def test_every_unit_counts_once(gpu_client, name, dtype):
    module, ins = ap.case(name, dtype)
    (got,), _ = run(gpu_client, module, ins, [dtype])
    want, tol = ap.wanted(module, ins, dtype)
    within(got, want, tol, name)
    assert not got[~want.any(axis=(1, 2))].any()


@pytest.mark.parametrize("name", ["long_one", "step_ragged", "ranges"])
def test_every_unit_counts_once_for_strided_queries(gpu_client, name):
    # queries as a slice of one projection, read in place
    whole, ins = ap.case(name, "bf16")
    x = op.values(ins)
    (t, hq, d), hkv = x[0].shape, x[1].shape[1]
    wide = np.random.RandomState(3).randn(t, hq + 2 * hkv, d)
    wide[:, hkv:hkv + hq] = x[0]
    a = op.host(wide, "bf16")
    ty = [f"tensor<{'x'.join(map(str, v.dims))}x{e}>" for v, e in zip([a] + ins[1:], ("bf16", "bf16", "bf16", "i32", "i32", "i32"))]
    q = f"tensor<{t}x{hq}x{d}xbf16>"
    call = operators.paged_attention("%o", [("%q", q)] + [(f"%x{i}", n) for i, n in enumerate(ty) if i], scale=d ** -0.5)
    module = (f"module {{\n  func.func @main({', '.join(f'%x{i}: {n}' for i, n in enumerate(ty))}) -> {q} {{\n"
              f"    %q = stablehlo.slice %x0 [0:{t}, {hkv}:{hkv + hq}, 0:{d}] : ({ty[0]}) -> {q}\n{call}    return %o : {q}\n  }}\n}}\n")
    (got,), _ = run(gpu_client, module, [a] + ins[1:], ["bf16"])
    want, tol = ap.wanted(whole, ins, "bf16")
    within(got, want, tol, name)
