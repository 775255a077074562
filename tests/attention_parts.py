"""Attention whose result shows every unit of 32 keys by itself, and how far a result may be from the oracle's, row by
row. The value of a key is 1 in one element, that of its unit (modulo the head dim), and 0 elsewhere (a sequence's last
key, which may be a unit alone, 16): an element of the output is the probability of its units, a few thousandths of the
whole over long contexts, and a unit that is lost, counted twice or given another weight moves it by a good part of
itself."""
from __future__ import annotations

import numpy as np

from oracle import operators as oo
from tests import operator_programs as op

UNIT = 32  # keys; no kernel's unit, block or range holds fewer, but a sequence's last


def _spread(n, most, seed):
    return [int(v) for v in np.random.RandomState(seed).randint(1, most + 1, n)]


CASES = {
    # decoding steps: stretches of units, joined by the workgroup that arrives last
    "step_mha": dict(new=[1] * 3, lengths=[500, 17, 1000], heads=(4, 4, 64), page=32),
    "step_one_head": dict(new=[1], lengths=[9001], heads=(2, 1, 64), page=16),
    "step_ragged": dict(new=[1] * 9, lengths=[4000, 1, 33, 2500, 64, 700, 65, 1300, 31], heads=(8, 2, 128), page=16),
    "step_many": dict(new=[1] * 70, lengths=[70 + 5 * i for i in range(70)], heads=(4, 2, 64), page=16),
    "step_verify": dict(new=[4, 1, 8, 3], lengths=[1100, 1, 88, 2700], heads=(8, 2, 128), page=16),
    "step_window": dict(new=[1, 2], lengths=[3000, 900], heads=(8, 2, 128), page=16, window=1000, slopes=True),
    "step_just_short": dict(new=[1], lengths=[16100], heads=(2, 1, 64), page=16),
    # few long sequences and chunks: ranges of keys, joined by a second launch
    "long_one": dict(new=[1], lengths=[20001], heads=(4, 1, 128), page=32),
    "long_group": dict(new=[1], lengths=[17000], heads=(8, 1, 128), page=16),
    "long_ragged": dict(new=[1, 1, 2], lengths=[17000, 40, 3000], heads=(4, 2, 64), page=16, softcap=30.0),
    "ranges": dict(new=[5], lengths=[6001], heads=(8, 1, 128), page=16),
    "ranges_ragged": dict(new=[17, 2, 20, 1], lengths=[5000, 300, 64, 2000], heads=(5, 1, 64), page=16),
    "ranges_window": dict(new=[33, 40], lengths=[3000, 2500], heads=(4, 2, 128), page=16, window=700, slopes=True),
    "ranges_not_causal": dict(new=[20, 3], lengths=[2000, 900], heads=(8, 2, 64), page=64, causal=False, softcap=30.0),
    "ranges_poison": dict(new=[20, 9], lengths=[2001, 1100], heads=(4, 1, 64), page=16, poison=True),
    "ranges_two_tiles": dict(new=[70], lengths=[4000], heads=(4, 1, 64), page=16),
    "ranges_70": dict(new=_spread(70, 9, 3), lengths=[9 + n for n in _spread(70, 800, 4)], heads=(8, 1, 64), page=16),
    # tiles alone
    "prompts": dict(new=_spread(34, 50, 5), lengths=[50 + n for n in _spread(34, 200, 6)], heads=(4, 4, 64), page=16),
    # the kernel for any type and head dim
    "any": dict(new=[1, 3], lengths=[3001, 90], heads=(4, 2, 80), page=16),
}


def case(name, dtype):
    """The module and the inputs of a case, its values as above."""
    c = dict(CASES[name])
    new, lengths, (hq, hkv, d), page = (c.pop(k) for k in ("new", "lengths", "heads", "page"))
    module, ins = op.attention_case(new, lengths, hq, hkv, d, page, dtype, seed=len(name), **c)
    vc, table = op.values(ins)[2], op.values(ins)[3]
    for b, n in enumerate(lengths):
        pos = np.arange(n)
        rows = table[b, pos // page], pos % page
        for h in range(hkv):
            v = np.zeros((n, d))
            v[pos, (pos // UNIT + 7 * h) % d] = 1.0
            v[-1:] *= 16.0
            vc[rows[0], h, rows[1]] = v
    ins[2] = op.host(vc, dtype)
    return module, ins


def rows(x, cfg):
    """(token, head, positions seen, probabilities, their scores, Σ|q||k| of each, values) of every query and head that
    sees a key, in float64."""
    q, kc, vc, table, starts, lengths = x[:6]
    slopes = x[6] if len(x) > 6 else None
    hq, d, hkv, size = q.shape[1], q.shape[2], kc.shape[1], kc.shape[2]
    scale, cap, window = float(np.float32(cfg.get("scale", d ** -0.5))), cfg.get("softcap", 0.0), int(cfg.get("window", 0))
    for b in range(lengths.shape[0]):
        length, s0, s1 = int(lengths[b]), int(starts[b]), int(starts[b + 1])
        page, at = table[b, np.arange(length) // size], np.arange(length) % size
        for t in range(s0, s1):
            pos = length - (s1 - t)
            first = max(0, pos - window + 1) if window else 0
            seen = np.arange(first, min(length, pos + 1) if cfg.get("causal", 1.0) else length)
            if seen.size == 0:
                continue
            for h in range(hq):
                k, v = (c[page[seen], h * hkv // hq, at[seen]] for c in (kc, vc))
                s = scale * (k @ q[t, h])
                s = cap * np.tanh(s / cap) if cap else s
                s = s if slopes is None else s + slopes[h] * (seen - pos)
                p = np.exp(s - s.max())
                yield t, h, seen, p / p.sum(), s, np.abs(k) @ np.abs(q[t, h]) * abs(scale), v


def bound(x, cfg, dtype):
    """How far a result may be from the exact one. With probabilities p_j, values v_j and o = Σ p_j v_j, relative errors e_j
    of the p_j move o by Σ p_j e_j (v_j - o). They are: where probabilities are held as two terms of 16 bits, half a step of
    half a step (f16: not under 2^-32 of the largest, its subnormal numbers' half step at the scale that they are held
    at); the score's, an f32
    sum of D products, and its multiples by f32 constants, each a few roundings of it, of the cap and of the bias; an
    exponential, 2^-21. Then f32 sums of n / 4 steps at most and a join's, and the result's own rounding: half a step of it, or
    of its type's subnormal numbers (f16; the others' may be zero)."""
    d, cap = x[0].shape[2], cfg.get("softcap", 0.0)
    half = op.HALF_STEP[dtype]
    tol = np.full(x[0].shape, 2.0 ** -25 if dtype == "f16" else 2.0 ** -126)
    for t, h, seen, p, s, mag, v in rows(x, cfg):
        o = p @ v
        e = (half ** 2 if dtype != "f32" else 0.0) + (d + 16) * 2.0 ** -24 * mag + 2.0 ** -22 * (2 * np.abs(s) + cap) + 2.0 ** -21
        if len(x) > 6:
            e = e + 2.0 ** -22 * np.abs(x[6][h]) * (seen[-1] - seen)
        small = 2.0 ** -32 * p.max() if dtype == "f16" else 0.0
        off = (p * e + small) @ np.abs(v - o)
        tol[t, h] += half * np.abs(o) + 1.02 * off + (seen.size / 4 + 192) * 2.0 ** -24 * (p @ np.abs(v))
    return tol


def wanted(module, ins, dtype):
    """The oracle's result and its bound."""
    x, cfg = op.values(ins), op.config_of(module)
    want, = oo.paged_attention(x, cfg)
    assert np.isfinite(want).all()
    return want, bound(x, cfg, dtype)


def lost_and_doubled(module, ins):
    """For each (token, head): (units seen, results with one of them lost, results with one of them doubled)."""
    x, cfg = op.values(ins), op.config_of(module)
    d = x[0].shape[2]
    for t, h, seen, p, _, _, v in rows(x, cfg):
        unit = seen // UNIT
        units = np.unique(unit)
        mass = np.array([[(p[unit == u]).sum()] for u in units])
        part = np.array([p[unit == u] @ v[unit == u] for u in units])
        o = p @ v
        with np.errstate(invalid="ignore", divide="ignore"):
            less = np.where(mass < 1 - 1e-12, (o - part) / (1 - mass), 0.0)
        yield t, h, units, less, (o + part) / (1 + mass)
