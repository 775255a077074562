"""Inputs of the decoding operators for the tests, raw and as oracle values, and a bytecode writer that knows their
custom_call. Every case is drawn from its own seed."""
from __future__ import annotations

import re
import struct

import numpy as np

from oracle import numerics
from oracle import stablehlo as sh
from ryft_amd import operators, pjrt
from ryft_amd.configs import HostInput
from tests import mlir_bytecode as mb

TYPE = {"bf16": pjrt.BufferType.BF16, "f16": pjrt.BufferType.F16, "f32": pjrt.BufferType.F32,
        "i32": pjrt.BufferType.S32}
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # relative: half of torch.finfo(t).eps


def host(x, dt):
    x = np.asarray(x, dtype=np.float64 if dt in sh.FLOAT else np.int64)
    return HostInput(np.ascontiguousarray(sh.to_raw(numerics.round_to(x, dt) if dt in sh.FLOAT else x, dt)), TYPE[dt], x.shape)


def values(inputs):
    names = {v: k for k, v in TYPE.items()}
    return [sh.from_raw(x.data, names[x.type]).reshape(x.dims) for x in inputs]


def append_case(tokens, hq, hkv, d, rot, page, pages, dtype, *, norm, interleaved, start=0, bad_slots=False,
                magnitude=1.0, seed=0):
    r = np.random.RandomState(seed)
    slots = r.permutation(pages * page)[:tokens]
    if bad_slots and tokens:
        slots[::3] = np.resize([-1, pages * page, 2 ** 31 - 1, -2 ** 31], slots[::3].shape)
    freq = 10000.0 ** (-np.arange(rot // 2) / max(1, rot // 2))
    cache = (pages, hkv, page, d)
    ins = [host(r.randn(tokens, hq, d), dtype), host(r.randn(tokens, hkv, d), dtype), host(r.randn(tokens, hkv, d), dtype),
           host(np.arange(start, start + tokens), "i32"), host(slots, "i32"), host(freq, "f32"), host(r.randn(*cache), dtype),
           host(r.randn(*cache), dtype)]
    if norm:
        ins += [host(1 + 0.1 * r.randn(d), dtype), host(1 + 0.1 * r.randn(d), dtype)]
    module = operators.rope_append_module(tokens=tokens, q_heads=hq, kv_heads=hkv, head_dim=d, rotary_dim=rot, pages=pages,
                                          page_size=page, dtype=dtype, norm=norm, eps=1e-5, interleaved=interleaved,
                                          magnitude=magnitude)
    return module, ins


def append_chain(steps, tokens=3, hq=4, hkv=2, d=64, page=16, pages=2, returns=None, aliased=True, extra="", seed=0):
    """`steps` appends of other tokens to one pair of caches, each over the one before. `returns`: results by name (%r0#0 ...),
    all queries and the last caches otherwise; `extra`: more lines."""
    r = np.random.RandomState(seed)
    q, k = f"tensor<{tokens}x{hq}x{d}xbf16>", f"tensor<{tokens}x{hkv}x{d}xbf16>"
    i, f, c = f"tensor<{tokens}xi32>", f"tensor<{d // 2}xf32>", f"tensor<{pages}x{hkv}x{page}x{d}xbf16>"
    last = steps - 1
    returns = returns or [f"%r{n}#0" for n in range(steps)] + [f"%r{last}#1", f"%r{last}#2"]
    kind = [q if n.endswith("#0") else c for n in returns]
    alias = {"kc": f"%r{last}#1", "vc": f"%r{last}#2"}
    params, ins, body = [("f", f), ("kc", c), ("vc", c)], [host(10000.0 ** (-np.arange(d // 2) / d), "f32")], ""
    ins += [host(r.randn(pages, hkv, page, d), "bf16") for _ in range(2)]
    slots = r.permutation(pages * page)
    for n in range(steps):
        params += [(f"q{n}", q), (f"k{n}", k), (f"v{n}", k), (f"p{n}", i), (f"s{n}", i)]
        ins += [host(r.randn(tokens, h, d), "bf16") for h in (hq, hkv, hkv)]
        ins += [host(r.randint(0, 1000, tokens), "i32"), host(slots[n * tokens:(n + 1) * tokens], "i32")]
        caches = ("%kc", "%vc") if n == 0 else (f"%r{n - 1}#1", f"%r{n - 1}#2")
        body += operators.rope_append(f"%r{n}", [(f"%q{n}", q), (f"%k{n}", k), (f"%v{n}", k), (f"%p{n}", i), (f"%s{n}", i), ("%f", f),
                                                 (caches[0], c), (caches[1], c)])
    head = ", ".join(f"%{n}: {t}" + (f" {{tf.aliasing_output = {returns.index(alias[n])} : i32}}"
                                     if aliased and alias.get(n) in returns else "") for n, t in params)
    types = ", ".join(kind)
    return (f"module {{\n  func.func @main({head}) -> ({types}) {{\n{body}{extra}    return {', '.join(returns)} : {types}\n  }}\n}}\n", ins)


def attention_case(new, lengths, hq, hkv, d, page, dtype, *, window=0, softcap=0.0, slopes=False, causal=True, spare=0,
                   bad_pages=False, poison=False, seed=0, spread=1.0):
    """`spare`: rows of q that belong to no sequence. bad_pages: a few table entries outside the cache. poison: what no
    query may see (rows past a sequence's end, unused pages) is NaN and infinite."""
    r = np.random.RandomState(seed)
    b, tokens = len(new), sum(new) + spare
    need = [max(0, -(-n // page)) for n in lengths]
    m, pages = max(need + [1]) + 1, sum(need) + 3
    order, table, at = r.permutation(pages), np.full((b, m), -1), 0
    kc, vc = r.randn(pages, hkv, page, d) * spread, r.randn(pages, hkv, page, d)
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    if poison:
        seen = np.zeros((pages, page), dtype=bool)
        for i, n in enumerate(lengths):
            for p in range(max(0, n)):
                seen[table[i, p // page], p % page] = True
        junk = np.resize([np.nan, np.inf, -np.inf], (pages, hkv, page, d))
        hide = ~seen[:, None, :, None] & np.ones((1, hkv, 1, d), dtype=bool)
        kc[hide], vc[hide] = junk[hide], junk[hide]
    if bad_pages:
        flat = table.reshape(-1)
        flat[::4] = np.resize([-1, pages, 2 ** 31 - 1, -2 ** 31], flat[::4].shape)
    ins = [host(r.randn(tokens, hq, d) * spread, dtype), host(kc, dtype), host(vc, dtype), host(table, "i32"),
           host(np.cumsum([0] + list(new)), "i32"), host(lengths, "i32")]
    if slopes:
        ins.append(host(2.0 ** (-8.0 * np.arange(1, hq + 1) / hq), "f32"))
    module = operators.paged_attention_module(
        tokens=tokens, sequences=b, q_heads=hq, kv_heads=hkv, head_dim=d, pages=pages, page_size=page,
        pages_per_sequence=m, dtype=dtype, scale=d ** -0.5, softcap=softcap, window=window, causal=causal, slopes=slopes)
    return module, ins


def sample_case(logits, dtype, temperature, top_k, top_p, min_p, uniform):
    logits = np.asarray(logits, dtype=np.float64)
    rows = logits.shape[0]
    full = lambda v: np.broadcast_to(np.asarray(v, dtype=np.float64), (rows,))  # noqa: E731
    ins = [host(logits, dtype), host(full(temperature), "f32"), host(full(top_k), "i32"), host(full(top_p), "f32"),
           host(full(min_p), "f32"), host(full(uniform), "f32")]
    return operators.sample_module(rows=rows, vocab=logits.shape[1], dtype=dtype), ins


def config_of(module):
    from oracle import operators as oo
    line = next(ln for ln in module.split("\n") if "custom_call" in ln)
    return oo.config(line)


class OperatorWriter(mb.Writer):
    """mlir_bytecode's writer with the attributes of a custom_call: strings, 32-bit floats, whole numbers, dictionaries."""

    def attr(self, spec):
        kind = spec[0]
        if kind == "string":
            return self.string_attr(spec[1])
        if kind == "f32":
            bits = struct.unpack("<I", struct.pack("<f", spec[1]))[0]
            return self.battr(mb.varint(9) + mb.varint(self.elem("f32")) + mb.svarint(bits))
        if kind == "int":
            return self.battr(mb.varint(8) + mb.varint(self.elem(spec[2])) + mb.svarint(spec[1]))
        if kind == "dict":
            data = mb.varint(1) + mb.varint(len(spec[1]))
            for k, v in spec[1].items():
                data += mb.varint(self.string_attr(k)) + mb.varint(self.attr(v))
            return self.battr(data)
        return super().attr(spec)


FIELDS = ["call_target_name", "has_side_effect", "backend_config", "api_version", "called_computations",
          "operand_layouts", "result_layouts", "output_operand_aliases"]


def to_bytecode(module, monkeypatch, order="sorted", **kw):
    """The module as MLIR bytecode, its custom_calls included."""
    plain = mb._parse_op

    def parse(lhs, name, rest):
        if name != "stablehlo.custom_call":
            return plain(lhs, name, rest)
        target, args, attrs, types = re.match(r"@([\w.]+)\((.*?)\) \{(.*)\} : (.*)$", rest).groups()
        cfg = {}
        for item in filter(None, re.search(r"backend_config = \{(.*?)\}", attrs).group(1).split(", ")):
            k, v = item.split(" = ")
            v, _, ty = v.partition(" : ")
            cfg[k] = ("bool", v == "true") if not ty else ("f32", float(v)) if ty == "f32" else ("int", int(v), ty)
        _, outs = mb._types_after_colon(types)
        return mb.Op(name, re.findall(r"%[\w#]+", args), mb._result_names(lhs), outs,
                     {"call_target_name": ("string", target), "backend_config": ("dict", cfg),
                      "api_version": ("int", 4, "i32")})

    monkeypatch.setattr(mb, "_parse_op", parse)
    monkeypatch.setitem(mb.SORTED, "stablehlo.custom_call", sorted(FIELDS))
    monkeypatch.setitem(mb.DECLARED, "stablehlo.custom_call", FIELDS)
    monkeypatch.setattr(mb, "REQUIRED", mb.REQUIRED | {"call_target_name"})
    monkeypatch.setattr(mb, "Writer", OperatorWriter)
    return mb.to_bytecode(module, order=order, **kw)
