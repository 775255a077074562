"""Oracle of the plugin's decoding operators (`custom_call @ryft.*`), in float64, row by row from their definitions.
Values as in oracle.stablehlo: float64 arrays holding exactly the operands' values, int64 integers; results unrounded."""
from __future__ import annotations

import math
import re

import numpy as np


def config(rest: str) -> dict:
    """backend_config = {name = value : type, ...} of a custom_call line."""
    m = re.search(r"backend_config\s*=\s*\{(.*?)\}", rest)
    out = {}
    for item in (m.group(1).split(",") if m and m.group(1).strip() else []):
        k, _, v = item.partition("=")
        v = v.split(":")[0].strip()
        if v.startswith("0x"):
            out[k.strip()] = float(np.uint32(int(v, 16)).view(np.float32))
        else:
            out[k.strip()] = {"true": 1.0, "false": 0.0, "": 1.0}.get(v) if v in ("true", "false", "") else float(v)
    return out


def _f32(x) -> float:
    return float(np.float32(x))  # (config values are held in 32 bits)


def rope_append(ops, cfg):
    q, k, v, positions, slots, freq, kc, vc = [o.copy() for o in ops[:8]]
    half = freq.shape[0]
    for x, w in ((q, 8), (k, 9)):
        if len(ops) > 8:
            ms = np.mean(np.square(x), axis=-1, keepdims=True)
            x[...] = x / np.sqrt(ms + _f32(cfg.get("eps", 1e-6))) * ops[w]
        for t in range(x.shape[0]):
            for i in range(half):
                a, b = (2 * i, 2 * i + 1) if cfg.get("interleaved") else (i, i + half)
                ang = float(positions[t]) * float(freq[i])
                c, s = (f(ang) * _f32(cfg.get("magnitude", 1.0)) for f in (math.cos, math.sin))
                xa, xb = x[t, :, a].copy(), x[t, :, b].copy()
                x[t, :, a], x[t, :, b] = xa * c - xb * s, xb * c + xa * s
    pages, _, size, _ = kc.shape
    for t, slot in enumerate(int(s) for s in slots):
        if 0 <= slot < pages * size:
            kc[slot // size, :, slot % size] = k[t]
            vc[slot // size, :, slot % size] = v[t]
    return [q, kc, vc]


def paged_attention(ops, cfg):
    q, kc, vc, table, starts, lengths = ops[:6]
    slopes = ops[6] if len(ops) > 6 else None
    out = np.zeros_like(q)
    tokens, hq, d = q.shape
    pages, hkv, size, _ = kc.shape
    cap, window = _f32(cfg.get("softcap", 0)), int(cfg.get("window", 0))
    scale = _f32(cfg["scale"]) if "scale" in cfg else 1.0 / math.sqrt(d)
    for b in range(lengths.shape[0]):
        s0, s1 = (min(max(int(s), 0), tokens) for s in starts[b:b + 2])
        length = min(max(int(lengths[b]), 0), table.shape[1] * size)
        pos = np.arange(length)
        page = table[b, pos // size] if length else np.zeros(0, dtype=np.int64)
        there = (page >= 0) & (page < pages)
        pos, page = pos[there], page[there]
        for t in range(s0, s1):
            at = length - (s1 - t)
            see = np.ones(pos.shape, dtype=bool)
            if cfg.get("causal", 1.0):
                see &= pos <= at
            if window:
                see &= at - pos < window
            if not see.any():
                continue
            for h in range(hq):
                ks = kc[page[see], h * hkv // hq, pos[see] % size]
                vs = vc[page[see], h * hkv // hq, pos[see] % size]
                s = scale * (ks @ q[t, h])
                if cap > 0:
                    s = cap * np.tanh(s / cap)
                if slopes is not None:
                    s = s + slopes[h] * (pos[see] - at)
                p = np.exp(s - s.max())
                out[t, h] = p @ vs / p.sum()
    return [out]


def sample(ops, _cfg):
    logits, temperature, top_k, top_p, min_p, uniform = ops
    tokens, logs = [], []
    for r in range(logits.shape[0]):
        x = np.where(np.isnan(logits[r]), -np.inf, logits[r])
        order = sorted((i for i in range(x.size) if x[i] > -np.inf), key=lambda i: (-x[i], i))
        if not order:
            tokens.append(-1)
            logs.append(-np.inf)
            continue
        best, t = x[order[0]], temperature[r]
        w = {i: 1.0 if x[i] == best else math.exp((x[i] - best) / t) if t > 0 else 0.0 for i in order}
        if not t > 0:
            order = order[:1]
        if 0 < top_k[r]:
            order = order[:int(top_k[r])]
        order = [i for n, i in enumerate(order) if n == 0 or w[i] >= min_p[r]]
        if top_p[r] < 1:
            total, before, kept = math.fsum(w[i] for i in order), 0.0, []
            for i in order:
                if kept and not before < top_p[r] * total:
                    break
                kept.append(i)
                before += w[i]
            order = kept
        total = math.fsum(w[i] for i in order)
        run, token = 0.0, None
        for i in sorted(order):
            run += w[i]
            if token is None and run > uniform[r] * total:
                token = i
        token = max(order) if token is None else token
        tokens.append(token)
        logs.append(math.log(w[token] / total))
    return [np.array(tokens, dtype=np.int64), np.array(logs)]


def tree_attention(ops, cfg):
    q, kc, vc, table, starts, lengths, visible = ops
    out = np.zeros_like(q)
    tokens, hq, d = q.shape
    pages, hkv, size, _ = kc.shape
    cap, window = _f32(cfg.get("softcap", 0)), int(cfg.get("window", 0))
    scale = _f32(cfg["scale"]) if "scale" in cfg else 1.0 / math.sqrt(d)
    for b in range(lengths.shape[0]):
        s0, s1 = (min(max(int(s), 0), tokens) for s in starts[b:b + 2])
        length = min(max(int(lengths[b]), 0), table.shape[1] * size)
        first = length - (s1 - s0)  # (below 0: the first nodes have no position)
        for t in range(s0, s1):
            nodes = [j for j in range(min(s1 - s0, 32 * visible.shape[1])) if int(visible[t, j // 32]) >> j % 32 & 1]
            at = first + len(nodes) - 1
            see = [p for p in range(first) if not window or at - p < window] + [first + j for j in nodes if first + j >= 0]
            see = [(int(table[b, p // size]), p % size) for p in see]
            see = [(page, row) for page, row in see if 0 <= page < pages]
            if not see:
                continue
            page, row = (np.array(a) for a in zip(*see))
            for h in range(hq):
                s = scale * (kc[page, h * hkv // hq, row] @ q[t, h])
                if cap > 0:
                    s = cap * np.tanh(s / cap)
                p = np.exp(s - s.max())
                out[t, h] = p @ vc[page, h * hkv // hq, row] / p.sum()
    return [out]


def tree_accept(ops, _cfg):
    tokens, parents, targets, slots, starts = ops[:5]
    caches = [c.copy() for c in ops[5:]]
    total = tokens.shape[0]
    counts, emitted, path = [], np.full(total, -1), np.full(total, -1)
    for b in range(starts.shape[0] - 1):
        s0, s1 = (min(max(int(s), 0), total) for s in starts[b:b + 2])
        nodes = [0] if s1 > s0 else []
        while nodes:
            at = nodes[-1]
            named = [c for c in range(at + 1, s1 - s0) if parents[s0 + c] == at and tokens[s0 + c] == targets[s0 + at]]
            if not named:
                break
            nodes.append(named[0])
        counts.append(len(nodes))
        moves = []
        for j, node in enumerate(nodes):
            emitted[s0 + j], path[s0 + j] = targets[s0 + node], node
            moves.append((int(slots[s0 + node]), int(slots[s0 + j])))
        for c in caches:
            pages, _, size, _ = c.shape
            inside = [(a, z) for a, z in moves if 0 <= a < pages * size and 0 <= z < pages * size]
            rows = [c[a // size, :, a % size].copy() for a, _ in inside]
            for (_, z), row in zip(inside, rows):
                c[z // size, :, z % size] = row
    return [np.array(counts, dtype=np.int64), emitted, path] + caches


def int4_matmul(ops, _cfg):
    x, weight, scale = ops[:3]
    n, half = weight.shape
    w = np.zeros((n, 2 * half))
    w[:, 0::2], w[:, 1::2] = weight % 16, weight // 16
    group = 2 * half // scale.shape[1]
    zero = np.repeat(ops[3], group, axis=1) if len(ops) > 3 else 8
    return [x @ ((w - zero) * np.repeat(scale, group, axis=1)).T]


OPERATORS = {"ryft.rope_append": rope_append, "ryft.paged_attention": paged_attention, "ryft.sample": sample,
             "ryft.tree_attention": tree_attention, "ryft.tree_accept": tree_accept, "ryft.int4_matmul": int4_matmul}
