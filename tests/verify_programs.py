"""Inputs of the operators that verify drafted tokens (tree_attention, tree_accept, int4_matmul) for the tests, raw and as
oracle values. Every case is drawn from its own seed."""
from __future__ import annotations

import numpy as np

from oracle import stablehlo as sh
from ryft_amd import operators, pjrt
from ryft_amd.configs import HostInput
from tests import operator_programs as op

TYPE = {**op.TYPE, "ui8": pjrt.BufferType.U8}


def host(x, dt):
    return HostInput(np.ascontiguousarray(np.asarray(x).astype(np.uint8)), TYPE[dt], np.shape(x)) if dt == "ui8" else op.host(x, dt)


def values(inputs):
    names = {v: k for k, v in TYPE.items()}
    return [sh.from_raw(x.data, names[x.type]).reshape(x.dims) for x in inputs]


def random_tree(n, r, wide=False):
    """Each node's parent: of all before it, or, for a deep tree, of the last three."""
    return [-1] + [int(r.randint(0 if wide else max(0, j - 3), j)) for j in range(1, n)]


def ancestor_words(parents, words):
    """Bits of each node's ancestors and itself."""
    out = np.zeros((len(parents), words), dtype=np.uint32)
    for j, p in enumerate(parents):
        if p >= 0:
            out[j] = out[p]
        if j < 32 * words:
            out[j, j // 32] |= np.uint32(1) << np.uint32(j % 32)
    return out.view(np.int32)


def tree_case(nodes, lengths, hq, hkv, d, page, dtype, *, words=None, window=0, softcap=0.0, spare=0, bad_pages=False, poison=False,
              masks="tree", seed=0, spread=1.0):
    """`masks`: "tree" (ancestors and itself), "random" (any nodes, those past a tree's end among them), "none" (no bits),
    "all". spare, bad_pages, poison as in operator_programs.attention_case."""
    r = np.random.RandomState(seed)
    _, ins = op.attention_case(nodes, lengths, hq, hkv, d, page, dtype, spare=spare, bad_pages=bad_pages, poison=poison, seed=seed,
                               spread=spread)
    words = words or max(1, -(-max(nodes) // 32))
    rows = []
    for n in nodes:
        if masks == "tree":
            rows.append(ancestor_words(random_tree(n, r, wide=True), words) if n else np.zeros((0, words), dtype=np.int32))
        else:
            bits = {"random": r.randint(-2 ** 31, 2 ** 31, (n, words)), "none": np.zeros((n, words)), "all": np.full((n, words), -1)}
            rows.append(bits[masks].astype(np.int32))
    rows.append(r.randint(-2 ** 31, 2 ** 31, (spare, words)).astype(np.int32))
    q, kc, _, table = ins[:4]
    module = operators.tree_attention_module(
        tokens=q.dims[0], sequences=len(nodes), q_heads=hq, kv_heads=hkv, head_dim=d, pages=kc.dims[0], page_size=page,
        pages_per_sequence=table.dims[1], words=words, dtype=dtype, scale=d ** -0.5, softcap=softcap, window=window)
    return module, ins + [host(np.concatenate(rows), "i32")]


def accept_case(nodes, caches, hkv, d, page, dtype, *, spare=0, bad_parents=False, bad_slots=False, vocab=3, wide=False, seed=0):
    """A small vocabulary, so that choices meet drafted tokens, equal siblings among them."""
    r = np.random.RandomState(seed)
    tokens = sum(nodes) + spare
    parents = np.array([p for n in nodes for p in random_tree(n, r, wide)[:n]] + [0] * spare, dtype=np.int64)
    if bad_parents and tokens:
        where = r.rand(tokens) < 0.15
        parents[where] = np.resize([-5, 2 ** 31 - 1, -2 ** 31, tokens, 70], int(where.sum()))
    pages = -(-tokens // page) + 2
    slots = r.permutation(pages * page)[:tokens]
    if bad_slots and tokens:
        slots[::4] = np.resize([-1, pages * page, 2 ** 31 - 1, -2 ** 31], slots[::4].shape)
    ins = [host(r.randint(0, vocab, tokens), "i32"), host(parents, "i32"), host(r.randint(0, vocab, tokens), "i32"), host(slots, "i32"),
           host(np.cumsum([0] + list(nodes)), "i32")]
    ins += [host(r.randn(pages, hkv, page, d), dtype) for _ in range(caches)]
    module = operators.tree_accept_module(tokens=tokens, sequences=len(nodes), caches=caches, pages=pages, kv_heads=hkv, page_size=page,
                                          head_dim=d, dtype=dtype)
    return module, ins


def int4_case(rows, k, n, group, dtype, *, zeros=False, scale_dtype=None, out_dtype=None, exact=False, seed=0):
    """`exact`: whole numbers and scales that are powers of two, so that every sum is exact in 32 bits."""
    r = np.random.RandomState(seed)
    groups = k // group
    if exact:
        x, scale = r.randint(-3, 4, (rows, k)), 2.0 ** r.randint(-2, 3, (n, groups))
    else:
        x, scale = r.randn(rows, k), r.uniform(0.002, 0.02, (n, groups))
    ins = [host(x, dtype), host(r.randint(0, 256, (n, k // 2)), "ui8"), host(scale, scale_dtype or dtype)]
    if zeros:
        ins.append(host(r.randint(0, 16, (n, groups)), "ui8"))
    return operators.int4_matmul_module(rows=rows, inner=k, columns=n, group=group, dtype=dtype, scale_dtype=scale_dtype,
                                        out_dtype=out_dtype, zeros=zeros), ins


def int4_error(x):
    """What f32 sums may be off by, for each element: a product with a weight, its zero point and a bias of 16 that the
    matrix kernels carry each have at most (q + z + 32) · scale · |x| behind them, and a sum passes through at most K / 32 +
    48 additions, each half a step of 2^-24 off: 32 within a matrix instruction, one for each of the K / 32 instructions,
    and those over lanes, wavefronts and ranges of K."""
    a, weight, scale = x[:3]
    n, half = weight.shape
    w = np.zeros((n, 2 * half))
    w[:, 0::2], w[:, 1::2] = weight % 16, weight // 16
    group = 2 * half // scale.shape[1]
    z = np.repeat(x[3], group, axis=1) if len(x) > 3 else 8
    return (2 * half / 32 + 48) * 2.0 ** -24 * (np.abs(a) @ ((w + z + 32) * np.repeat(np.abs(scale), group, axis=1)).T)
