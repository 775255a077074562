"""Programs for the plugin's decoding operators: `stablehlo.custom_call @ryft.<name>` in its typed form (api_version 4,
a `backend_config` dictionary), as MLIR text for `Program.mlir`.

Operators (operands → results; T tokens, B sequences, Hq / Hkv query / key heads of D values; cache types and q, k, v
are one of bf16, f16, f32):

* ``ryft.rope_append`` (q [T,Hq,D], k [T,Hkv,D], v [T,Hkv,D], positions [T] i32, slots [T] i32, inv_freq [R/2] f32,
  k_cache, v_cache [pages,Hkv,page_size,D] (, q_weight, k_weight [D])) → (q [T,Hq,D], k_cache, v_cache).
  RMSNorm of every query and key head where there are weights (`eps`), the first R values of each turned by position ·
  inv_freq (pairs i and i + R/2, or 2i and 2i + 1 with `interleaved`), cosine and sine times `magnitude`; keys and values
  written to slot = page · page_size + row. A slot outside the cache is not written; slots of a call are distinct.
* ``ryft.paged_attention`` (q [T,Hq,D], k_cache, v_cache, page_table [B,M] i32, starts [B+1] i32, lengths [B] i32
  (, slopes [Hq] f32)) → o [T,Hq,D]. Sequence b's queries are rows starts[b] .. starts[b+1]-1 of q, the last of its
  lengths[b] positions; the key of position p is row p % page_size of page page_table[b][p / page_size]. Scores are
  scale · q·k, capped to softcap · tanh(s / softcap) if `softcap` > 0, plus slopes[h] · (key - query position); a query
  sees the keys up to itself (`causal`), the last `window` of them if `window` > 0, and none on a page outside the cache.
  A query that sees nothing, or belongs to no sequence, gets zeros. starts do not decrease.
* ``ryft.sample`` (logits [B,V], temperature [B] f32, top_k [B] i32, top_p, min_p, uniform [B] f32) → (token [B] i32,
  logprob [B] f32). The softmax of logits / temperature, computed in 64 bits, cut to the top_k largest (0: all; of equal
  logits the lower index first), to those of at least min_p times the largest, and to the smallest prefix of what is
  left, in falling order, that holds top_p of its weight; the token is where the running sum of what is kept, by index,
  passes uniform (in [0, 1)) of the total. temperature 0 takes the largest; the largest is always kept (of several, by a
  min_p above 1, the first alone); a NaN logit is never drawn; a row with no logit above -inf gives token -1 and logprob
  -inf.

The caches are results as well as operands. With `tf.aliasing_output` on the parameters (the modules below have it) and a
donated argument, or the same address as parameter and result of `execute_into`, only the new tokens are written;
otherwise the cache is copied first. Appends to one cache after each other write one buffer where each is all that reads
the caches of the one before; a cache between two appends that an attention reads, or that is a result, is copied.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import numpy as np


def _t(shape, dtype: str) -> str:
    return "tensor<" + "".join(f"{d}x" for d in shape) + dtype + ">"


def _f32(x: float) -> str:
    x = np.float32(x)
    if not np.isfinite(x):
        return f"0x{x.view(np.uint32):08X} : f32"
    return np.format_float_scientific(x, unique=True, exp_digits=2) + " : f32"


def _call(results: Sequence[str], target: str, operands: Sequence[Tuple[str, str]], types: Sequence[str], config) -> str:
    """One custom_call line: result names, (operand name, type) pairs, result types, config entries as text."""
    names = results[0].split("#")[0] if len(results) > 1 else results[0]
    head = f"{names}:{len(results)}" if len(results) > 1 else names
    cfg = ", ".join(f"{k} = {v}" for k, v in config)
    outs = types[0] if len(types) == 1 else "(" + ", ".join(types) + ")"
    return (f"    {head} = stablehlo.custom_call @{target}({', '.join(n for n, _ in operands)}) {{api_version = 4 : i32, "
            f"backend_config = {{{cfg}}}}} : ({', '.join(t for _, t in operands)}) -> {outs}\n")


def rope_append(result: str, operands: Sequence[Tuple[str, str]], *, eps: Optional[float] = None,
                interleaved: bool = False, magnitude: float = 1.0) -> str:
    """The line `result:3 = custom_call @ryft.rope_append(...)`; its results are result#0 (q), #1 and #2 (the caches)."""
    cfg = [("interleaved", "true" if interleaved else "false"), ("magnitude", _f32(magnitude))]
    if eps is not None:
        cfg.append(("eps", _f32(eps)))
    q, kc, vc = operands[0][1], operands[6][1], operands[7][1]
    return _call([f"{result}#{i}" for i in range(3)], "ryft.rope_append", operands, [q, kc, vc], cfg)


def paged_attention(result: str, operands: Sequence[Tuple[str, str]], *, scale: float, softcap: float = 0.0,
                    window: int = 0, causal: bool = True) -> str:
    """The line `result = custom_call @ryft.paged_attention(...)`."""
    cfg = [("causal", "true" if causal else "false"), ("scale", _f32(scale)), ("softcap", _f32(softcap)),
           ("window", f"{int(window)} : i64")]
    return _call([result], "ryft.paged_attention", operands, [operands[0][1]], cfg)


def sample(result: str, operands: Sequence[Tuple[str, str]], rows: int) -> str:
    """The line `result:2 = custom_call @ryft.sample(...)`; its results are result#0 (token) and result#1 (logprob)."""
    return _call([f"{result}#0", f"{result}#1"], "ryft.sample", operands, [_t((rows,), "i32"), _t((rows,), "f32")], [])


def rope_append_module(*, tokens: int, q_heads: int, kv_heads: int, head_dim: int, rotary_dim: int, pages: int,
                       page_size: int, dtype: str = "bf16", norm: bool = False, eps: float = 1e-6,
                       interleaved: bool = False, magnitude: float = 1.0) -> str:
    """A module of one rope_append: its operands are the parameters, both caches aliased to their results."""
    q, k = _t((tokens, q_heads, head_dim), dtype), _t((tokens, kv_heads, head_dim), dtype)
    i, f = _t((tokens,), "i32"), _t((rotary_dim // 2,), "f32")
    c, w = _t((pages, kv_heads, page_size, head_dim), dtype), _t((head_dim,), dtype)
    types = [q, k, k, i, i, f, c, c] + ([w, w] if norm else [])
    alias = {6: 1, 7: 2}
    params = ", ".join(f"%arg{n}: {t}" + (f" {{tf.aliasing_output = {alias[n]} : i32}}" if n in alias else "")
                       for n, t in enumerate(types))
    call = rope_append("%0", [(f"%arg{n}", t) for n, t in enumerate(types)], eps=eps if norm else None,
                       interleaved=interleaved, magnitude=magnitude)
    return f"module {{\n  func.func @main({params}) -> ({q}, {c}, {c}) {{\n{call}    return %0#0, %0#1, %0#2 : {q}, {c}, {c}\n  }}\n}}\n"


def paged_attention_module(*, tokens: int, sequences: int, q_heads: int, kv_heads: int, head_dim: int, pages: int,
                           page_size: int, pages_per_sequence: int, dtype: str = "bf16", scale: float,
                           softcap: float = 0.0, window: int = 0, causal: bool = True, slopes: bool = False) -> str:
    """A module of one paged_attention: its operands are the parameters."""
    q, c = _t((tokens, q_heads, head_dim), dtype), _t((pages, kv_heads, page_size, head_dim), dtype)
    types = [q, c, c, _t((sequences, pages_per_sequence), "i32"), _t((sequences + 1,), "i32"), _t((sequences,), "i32")]
    types += [_t((q_heads,), "f32")] if slopes else []
    params = ", ".join(f"%arg{n}: {t}" for n, t in enumerate(types))
    call = paged_attention("%0", [(f"%arg{n}", t) for n, t in enumerate(types)], scale=scale, softcap=softcap,
                           window=window, causal=causal)
    return f"module {{\n  func.func @main({params}) -> {q} {{\n{call}    return %0 : {q}\n  }}\n}}\n"


def sample_module(*, rows: int, vocab: int, dtype: str = "f32") -> str:
    """A module of one sample: its operands are the parameters."""
    f, i = _t((rows,), "f32"), _t((rows,), "i32")
    types = [_t((rows, vocab), dtype), f, i, f, f, f]
    params = ", ".join(f"%arg{n}: {t}" for n, t in enumerate(types))
    call = sample("%0", [(f"%arg{n}", t) for n, t in enumerate(types)], rows)
    return f"module {{\n  func.func @main({params}) -> ({i}, {f}) {{\n{call}    return %0#0, %0#1 : {i}, {f}\n  }}\n}}\n"


def _rms_norm(p: str, x: str, w: str, rows: int, d: int, eps: float) -> str:
    """%<p>n = RMSNorm(x)·w in bf16, the form the row-norm kernels recognise."""
    xt, wt, xf, rf, wf = _t((rows, d), "bf16"), _t((d,), "bf16"), _t((rows, d), "f32"), _t((rows,), "f32"), _t((d,), "f32")
    lit = lambda v: np.format_float_scientific(np.float32(v), unique=True, exp_digits=2)  # noqa: E731
    return f"""    %{p}0 = stablehlo.convert {x} : ({xt}) -> {xf}
    %{p}1 = stablehlo.multiply %{p}0, %{p}0 : {xf}
    %{p}z = stablehlo.constant dense<0.000000e+00> : tensor<f32>
    %{p}2 = stablehlo.reduce(%{p}1 init: %{p}z) applies stablehlo.add across dimensions = [1] : ({xf}, tensor<f32>) -> {rf}
    %{p}a = stablehlo.constant dense<{lit(1.0 / d)}> : tensor<f32>
    %{p}3 = stablehlo.broadcast_in_dim %{p}a, dims = [] : (tensor<f32>) -> {rf}
    %{p}4 = stablehlo.multiply %{p}2, %{p}3 : {rf}
    %{p}e = stablehlo.constant dense<{lit(eps)}> : tensor<f32>
    %{p}5 = stablehlo.broadcast_in_dim %{p}e, dims = [] : (tensor<f32>) -> {rf}
    %{p}6 = stablehlo.add %{p}4, %{p}5 : {rf}
    %{p}7 = stablehlo.rsqrt %{p}6 : {rf}
    %{p}8 = stablehlo.broadcast_in_dim %{p}7, dims = [0] : ({rf}) -> {xf}
    %{p}9 = stablehlo.multiply %{p}0, %{p}8 : {xf}
    %{p}w = stablehlo.convert {w} : ({wt}) -> {wf}
    %{p}x = stablehlo.broadcast_in_dim %{p}w, dims = [1] : ({wf}) -> {xf}
    %{p}y = stablehlo.multiply %{p}9, %{p}x : {xf}
    %{p}n = stablehlo.convert %{p}y : ({xf}) -> {xt}
"""


def _dot(r: str, a: str, b: str, m: int, k: int, n: int, contract: str = "[1] x [0]", rhs: Optional[str] = None) -> str:
    """%<r> = a [m,k] · b [k,n], f32."""
    return (f"    %{r} = stablehlo.dot_general {a}, {b}, contracting_dims = {contract} : ({_t((m, k), 'bf16')}, "
            f"{rhs or _t((k, n), 'bf16')}) -> {_t((m, n), 'f32')}\n")


def _rows(r: str, table: str, index: str, rows: int, d: int, n: int) -> str:
    """%<r> = rows `index` [n] of `table` [rows, d]."""
    return (f'    %{r} = "stablehlo.gather"({table}, {index}) <{{dimension_numbers = #stablehlo.gather<offset_dims = [1], '
            f"collapsed_slice_dims = [0], start_index_map = [0], index_vector_dim = 1>, indices_are_sorted = false, "
            f"slice_sizes = array<i64: 1, {d}>}}> : ({_t((rows, d), 'bf16')}, {_t((n,), 'i32')}) -> {_t((n, d), 'bf16')}\n")


def decoder_module(*, tokens: int, sequences: int, vocab: int, layers: int, d_model: int, q_heads: int, kv_heads: int,
                   head_dim: int, ffn: int, pages: int, page_size: int, pages_per_sequence: int, eps: float = 1e-6,
                   softcap: float = 0.0, window: int = 0) -> Tuple[str, List[Tuple[str, Tuple[int, ...], str]]]:
    """One step of a small bf16 decoder over a ragged batch, prompts and single tokens alike: embedding rows, per layer
    RMSNorm, a fused query/key/value projection, rope_append, paged_attention, output projection and a SwiGLU block,
    then the norm and the tied output projection of each sequence's last token (`last`), and sample. Returns the module
    and its parameters as (name, shape, element type); its results are the tokens, their log-probabilities, and every
    layer's caches, aliased to their parameters."""
    t, b, hd = tokens, sequences, head_dim
    wide = (q_heads + 2 * kv_heads) * hd
    cache = (pages, kv_heads, page_size, hd)
    params: List[Tuple[str, Tuple[int, ...], str]] = [
        ("ids", (t,), "i32"), ("positions", (t,), "i32"), ("slots", (t,), "i32"),
        ("table", (b, pages_per_sequence), "i32"), ("starts", (b + 1,), "i32"), ("lengths", (b,), "i32"),
        ("last", (b,), "i32"), ("temperature", (b,), "f32"), ("top_k", (b,), "i32"), ("top_p", (b,), "f32"),
        ("min_p", (b,), "f32"), ("uniform", (b,), "f32"), ("inv_freq", (hd // 2,), "f32"),
        ("embed", (vocab, d_model), "bf16"), ("norm", (d_model,), "bf16")]
    for n in range(layers):
        params += [(f"l{n}_norm1", (d_model,), "bf16"), (f"l{n}_qkv", (d_model, wide), "bf16"),
                   (f"l{n}_qw", (hd,), "bf16"), (f"l{n}_kw", (hd,), "bf16"), (f"l{n}_o", (q_heads * hd, d_model), "bf16"),
                   (f"l{n}_norm2", (d_model,), "bf16"), (f"l{n}_gate_up", (d_model, 2 * ffn), "bf16"),
                   (f"l{n}_down", (ffn, d_model), "bf16"),
                   (f"l{n}_k", cache, "bf16"), (f"l{n}_v", cache, "bf16")]
    types = {name: _t(shape, dt) for name, shape, dt in params}
    xt, xf, q3, k3, qt = _t((t, d_model), "bf16"), _t((t, d_model), "f32"), _t((t, q_heads, hd), "bf16"), \
        _t((t, kv_heads, hd), "bf16"), _t((t, q_heads * hd), "bf16")
    a3, wt, wf, ht, hf = _t((t, q_heads + 2 * kv_heads, hd), "bf16"), _t((t, wide), "bf16"), _t((t, wide), "f32"), \
        _t((t, ffn), "bf16"), _t((t, ffn), "f32")
    arg = lambda n: (f"%{n}", types[n])  # noqa: E731
    body = _rows("x", "%embed", "%ids", vocab, d_model, t)
    x = "%x"
    caches = []
    for n in range(layers):
        p = f"l{n}"
        body += _rms_norm(f"{p}a", x, f"%{p}_norm1", t, d_model, eps)
        body += _dot(f"{p}p", f"%{p}an", f"%{p}_qkv", t, d_model, wide)
        body += f"    %{p}pb = stablehlo.convert %{p}p : ({wf}) -> {wt}\n"
        body += f"    %{p}ph = stablehlo.reshape %{p}pb : ({wt}) -> {a3}\n"
        for name, lo, hi, ty in (("q", 0, q_heads, q3), ("k", q_heads, q_heads + kv_heads, k3),
                                 ("v", q_heads + kv_heads, q_heads + 2 * kv_heads, k3)):
            body += f"    %{p}{name} = stablehlo.slice %{p}ph [0:{t}, {lo}:{hi}, 0:{hd}] : ({a3}) -> {ty}\n"
        body += rope_append(f"%{p}r", [(f"%{p}q", q3), (f"%{p}k", k3), (f"%{p}v", k3), arg("positions"), arg("slots"),
                                       arg("inv_freq"), arg(f"{p}_k"), arg(f"{p}_v"), arg(f"{p}_qw"), arg(f"{p}_kw")], eps=eps)
        ct = types[f"{p}_k"]
        body += paged_attention(f"%{p}t", [(f"%{p}r#0", q3), (f"%{p}r#1", ct), (f"%{p}r#2", ct), arg("table"),
                                           arg("starts"), arg("lengths")], scale=hd ** -0.5, softcap=softcap, window=window)
        caches += [f"%{p}r#1", f"%{p}r#2"]
        body += f"    %{p}u = stablehlo.reshape %{p}t : ({q3}) -> {qt}\n"
        body += _dot(f"{p}w", f"%{p}u", f"%{p}_o", t, q_heads * hd, d_model)
        body += f"    %{p}xf = stablehlo.convert {x} : ({xt}) -> {xf}\n"
        body += f"    %{p}s = stablehlo.add %{p}xf, %{p}w : {xf}\n    %{p}sb = stablehlo.convert %{p}s : ({xf}) -> {xt}\n"
        body += _rms_norm(f"{p}b", f"%{p}sb", f"%{p}_norm2", t, d_model, eps)
        body += _dot(f"{p}gu", f"%{p}bn", f"%{p}_gate_up", t, d_model, 2 * ffn)
        for name, lo, hi in (("g", 0, ffn), ("h", ffn, 2 * ffn)):
            body += f"    %{p}{name} = stablehlo.slice %{p}gu [0:{t}, {lo}:{hi}] : ({_t((t, 2 * ffn), 'f32')}) -> {hf}\n"
        body += f"    %{p}i = stablehlo.logistic %{p}g : {hf}\n    %{p}j = stablehlo.multiply %{p}g, %{p}i : {hf}\n"
        body += f"    %{p}m = stablehlo.multiply %{p}j, %{p}h : {hf}\n    %{p}mb = stablehlo.convert %{p}m : ({hf}) -> {ht}\n"
        body += _dot(f"{p}d", f"%{p}mb", f"%{p}_down", t, ffn, d_model)
        body += f"    %{p}sf = stablehlo.convert %{p}sb : ({xt}) -> {xf}\n"
        body += f"    %{p}y = stablehlo.add %{p}sf, %{p}d : {xf}\n    %{p}yb = stablehlo.convert %{p}y : ({xf}) -> {xt}\n"
        x = f"%{p}yb"
    body += _rows("z", x, "%last", t, d_model, b)
    body += _rms_norm("f", "%z", "%norm", b, d_model, eps)
    body += _dot("logits", "%fn", "%embed", b, d_model, vocab, "[1] x [1]", types["embed"])
    body += sample("%out", [("%logits", _t((b, vocab), "f32"))] + [arg(n) for n in ("temperature", "top_k", "top_p", "min_p", "uniform")], b)
    outs = [_t((b,), "i32"), _t((b,), "f32")] + [types[f"l{n}_k"] for n in range(layers) for _ in range(2)]
    alias = {f"l{n}_{c}": 2 + 2 * n + i for n in range(layers) for i, c in enumerate("kv")}
    head = ", ".join(f"%{n}: {types[n]}" + (f" {{tf.aliasing_output = {alias[n]} : i32}}" if n in alias else "") for n, _, _ in params)
    rets = ", ".join(["%out#0", "%out#1"] + caches)
    return (f"module {{\n  func.func @main({head}) -> ({', '.join(outs)}) {{\n{body}    return {rets} : {', '.join(outs)}\n  }}\n}}\n",
            params)
