"""The oracle's bound of attention_parts.py on the CPU: it leaves no room for a unit of 32 keys that is lost or counted
twice, nor for a result of zeros, or (bf16) of probabilities of one 16-bit term, and holds the oracle's own result with its
probabilities as two."""
import numpy as np
import pytest

from oracle import numerics
from tests import attention_parts as ap
from tests import operator_programs as op


@pytest.mark.parametrize("name, dtype", [(n, "bf16") for n in ap.CASES] + [(n, "f16") for n in ("step_one_head", "ranges_window")])
def test_the_bound_shows_every_unit(name, dtype):
    module, ins = ap.case(name, dtype)
    want, tol = ap.wanted(module, ins, dtype)
    seen = want.any(axis=2)
    assert (np.abs(want) > tol).any(axis=2)[seen].all()              # (zeros)
    missed = {}
    for t, h, units, less, more in ap.lost_and_doubled(module, ins):
        if units.size == 1:  # (doubled alone it is itself)
            more = less
        for result in (less, more):
            for u, row in zip(units, result):
                found = (np.abs(row - want[t, h]) > tol[t, h]).any()
                missed[t, u] = missed.get((t, u), True) and not found
    # of every query, by at least one of its heads; far units of a steep bias have no weight in any
    weight = {}
    x, cfg = op.values(ins), op.config_of(module)
    for t, h, s, p, *_ in ap.rows(x, cfg):
        for u in np.unique(s // ap.UNIT):
            weight[t, u] = max(weight.get((t, u), 0.0), p[s // ap.UNIT == u].sum())
    left = {k for k, v in missed.items() if v and weight[k] > (2e-3 if len(x) > 6 else 0.0)}
    assert not left, (len(left), len(missed), sorted(left)[:5])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["step_verify", "step_many", "ranges_window", "ranges_70"])
def test_the_bound_holds_probabilities_in_two_terms(name, dtype):
    module, ins = ap.case(name, dtype)
    want, tol = ap.wanted(module, ins, dtype)
    one_term = 0
    for t, h, _, p, _, _, v in ap.rows(op.values(ins), op.config_of(module)):
        p = p / p.max() * 128
        first = numerics.round_to(p, dtype)
        both = first + numerics.round_to(p - first, dtype)
        got = numerics.round_to(both @ v / p.sum(), dtype)
        assert np.all(np.abs(got - want[t, h]) <= tol[t, h])
        one_term += not np.all(np.abs(numerics.round_to(first @ v / first.sum(), dtype) - want[t, h]) <= tol[t, h])
    assert one_term or dtype == "f16"
