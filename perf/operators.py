"""Timed operators of a decoding step: the rotary embedding that writes a paged cache, the attention that reads that
cache, and the sampler that turns logits into tokens. Each has a plain form of elementary torch operations (`own`
false) and the plugin's form (`own` true): a module with the operator's `stablehlo.custom_call`, compiled once, run on
the caller's device memory and stream.

Families (`family` of a case):

* ``append``    queries, keys and values of new tokens: RMSNorm of every query and key head, rotation by position
                (half or interleaved layout, whole head or its first part), keys and values written to their slots of
                a paged cache. Results: the queries, and both caches.
* ``attention`` queries of several sequences against their pages of the cache: grouped heads, causal, optionally with
                a window, scores capped by a tanh, or a bias that grows with distance.
* ``sample``    a token for each row of logits: temperature, top-k, top-p and min-p, the uniform number given.
                Results: the token and its log-probability.
"""
from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

# --------------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one new token of one sequence: the smallest call, bounded by latency
        dict(name="append_one", family="append", tokens=1, hq=32, hkv=8, d=128, rot=128, dtype="bf16", page=16,
             pages=64, norm=True, interleaved=False, start=4000, factor=1.0),
        # a decoding step of 256 sequences
        dict(name="append_decode", family="append", tokens=256, hq=32, hkv=8, d=128, rot=128, dtype="bf16", page=16,
             pages=1024, norm=True, interleaved=False, start=20000, factor=8.0),
        # prompts of 8192 tokens together, half of each head rotated in pairs of neighbours
        dict(name="append_prompt", family="append", tokens=8192, hq=32, hkv=8, d=128, rot=64, dtype="bf16", page=64,
             pages=160, norm=False, interleaved=True, start=0, factor=1.0),
        # a prompt of an odd length at far positions, heads of 64, f16
        dict(name="append_ragged", family="append", tokens=1777, hq=12, hkv=12, d=64, rot=64, dtype="f16", page=16,
             pages=150, norm=True, interleaved=False, start=900000, factor=32.0),
        # one query of one short sequence: the smallest call
        dict(name="attention_one", family="attention", sequences=1, new=1, context=500, ragged=False, hq=8, hkv=8,
             d=64, dtype="bf16", page=16, window=0, softcap=0.0, slopes=False),
        # a decoding step of 64 sequences of all lengths
        dict(name="attention_decode", family="attention", sequences=64, new=1, context=4096, ragged=True, hq=32, hkv=8,
             d=128, dtype="bf16", page=16, window=0, softcap=0.0, slopes=False),
        # two long sequences, capped scores: the key axis is all the parallelism there is
        dict(name="attention_long", family="attention", sequences=2, new=1, context=100001, ragged=False, hq=16,
             hkv=2, d=128, dtype="f16", page=32, window=0, softcap=30.0, slopes=False),
        # four prompts of up to 2048 tokens in one ragged batch
        dict(name="attention_prompt", family="attention", sequences=4, new=2048, context=2048, ragged=True, hq=32,
             hkv=8, d=128, dtype="bf16", page=16, window=0, softcap=50.0, slopes=False),
        # the next 512 tokens of two long prompts, with a window and a bias by distance
        dict(name="attention_chunk", family="attention", sequences=2, new=512, context=12000, ragged=True, hq=16,
             hkv=4, d=64, dtype="bf16", page=64, window=4096, softcap=0.0, slopes=True),
        # one row of logits: the smallest call
        dict(name="sample_one", family="sample", rows=1, vocab=32000, dtype="f32", filters="all"),
        # a decoding step of 64 sequences, each with settings of its own
        dict(name="sample_batch", family="sample", rows=64, vocab=128256, dtype="f32", filters="mixed"),
        # 256 rows of 16-bit logits, temperature alone
        dict(name="sample_plain", family="sample", rows=256, vocab=50257, dtype="bf16", filters="none"),
    ]


def _size(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; odd ones as likely as even ones."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.choice(["append", "attention", "attention", "sample"])
    hkv, group = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 2, 4, 5, 8])
    d, dtype, page = rng.choice([64, 128]), rng.choice(["bf16", "bf16", "f16"]), rng.choice([16, 32, 64, 128])
    if family == "append":
        tokens = _size(rng, 1, 8192)
        while tokens * (group + 2) * hkv * d > 1 << 25:
            tokens //= 2
        return dict(family="append", tokens=tokens, hq=hkv * group, hkv=hkv, d=d, rot=rng.choice([d, d, d // 2, d // 4]),
                    dtype=dtype, page=page, pages=-(-tokens // page) + rng.randint(1, 64), norm=rng.random() < 0.6,
                    interleaved=rng.random() < 0.4, start=rng.choice([0, _size(rng, 1, 1000000)]),
                    factor=rng.choice([1.0, 1.0, 8.0, 32.0]))
    if family == "attention":
        mode = rng.choice(["decode", "decode", "few", "prompt", "chunk"])
        while True:
            b = _size(rng, 1, 128)
            new = 1 if mode == "decode" else rng.randint(2, 8) if mode == "few" else _size(rng, 16, 2048)
            context = new if mode == "prompt" else new + _size(rng, 16, 65536)
            if b * hkv * group * new * context <= 1 << 28 and b * context * hkv * d <= 1 << 28:
                return dict(family="attention", sequences=b, new=new, context=context, ragged=rng.random() < 0.7,
                            hq=hkv * group, hkv=hkv, d=d, dtype=dtype, page=page,
                            window=rng.choice([0, 0, _size(rng, 64, 8192)]), softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                            slopes=rng.random() < 0.25)
    while True:
        rows, vocab = _size(rng, 1, 512), _size(rng, 1000, 262144)
        if rows * vocab <= 1 << 23:
            return dict(family="sample", rows=rows, vocab=vocab, dtype=rng.choice(["f32", "bf16", "f16"]),
                        filters=rng.choice(["none", "mixed", "all"]))


_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _lengths(c):
    """New tokens and total length of each sequence of an attention case: spread evenly where they differ."""
    new, total = [], []
    for i in range(c["sequences"]):
        f, g = ((i + 1) * 0.6180339887) % 1.0, ((i + 1) * 0.7548776662) % 1.0
        n = max(1, math.ceil(c["new"] * (0.25 + 0.75 * f))) if c["ragged"] else c["new"]
        prior = c["context"] - c["new"]
        new.append(n)
        total.append(n + (int(prior * g) if c["ragged"] else prior))
    return new, total


# --------------------------------------------------------------------------------------------------- inputs


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(shape, std=1.0, mean=0.0, dtype=None):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype or dt)

    def uniform(shape, lo, hi):
        return torch.rand(shape, generator=g, device="cuda").mul_(hi - lo).add_(lo)

    dt = _DTYPE[c["dtype"]]
    if c["family"] == "append":
        t, d = c["tokens"], c["d"]
        slots = torch.randperm(c["pages"] * c["page"], generator=g, device="cuda")[:t].to(torch.int32)
        freq = 500000.0 ** (-torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64) / (c["rot"] // 2))
        freq[c["rot"] // 4:] /= c["factor"]  # the slow half stretched for a longer context
        cache = (c["pages"], c["hkv"], c["page"], d)
        x = {"q": normal((t, c["hq"], d)), "k": normal((t, c["hkv"], d)), "v": normal((t, c["hkv"], d)),
             "positions": torch.arange(c["start"], c["start"] + t, device="cuda", dtype=torch.int32), "slots": slots,
             "freq": freq.float(), "k_cache": normal(cache), "v_cache": normal(cache)}
        if c["norm"]:
            x["q_weight"], x["k_weight"] = normal((d,), 0.1, 1.0), normal((d,), 0.1, 1.0)
        return x
    if c["family"] == "attention":
        new, total = _lengths(c)
        page, d = c["page"], c["d"]
        need = [-(-n // page) for n in total]
        pages = sum(need) + 7
        order = torch.randperm(pages, generator=g, device="cuda").cpu()  # (pages are handed out in no order)
        table, at = torch.full((c["sequences"], -(-c["context"] // page)), -1, dtype=torch.int32), 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        cache = (pages, c["hkv"], page, d)
        x = {"q": normal((sum(new), c["hq"], d), 1.5), "k_cache": normal(cache), "v_cache": normal(cache),
             "table": table.cuda(), "starts": torch.tensor(np.cumsum([0] + new), dtype=torch.int32).cuda(),
             "lengths": torch.tensor(total, dtype=torch.int32).cuda()}
        if c["slopes"]:
            x["slopes"] = torch.exp2(-8.0 * torch.arange(1, c["hq"] + 1, device="cuda") / c["hq"]).float()
        return x
    rows = c["rows"]
    x = {"logits": normal((rows, c["vocab"]), 3.0), "temperature": torch.ones(rows, device="cuda"),
         "top_k": torch.zeros(rows, device="cuda", dtype=torch.int32), "top_p": torch.ones(rows, device="cuda"),
         "min_p": torch.zeros(rows, device="cuda"), "uniform": uniform((rows,), 0.0, 1.0).clamp_(max=1.0 - 2.0 ** -24)}
    x["temperature"] = uniform((rows,), 0.5, 1.3)
    if c["filters"] != "none":
        kind = torch.arange(rows, device="cuda") % 5 if c["filters"] == "mixed" else torch.full((rows,), 5, device="cuda")
        x["top_k"] = torch.where((kind == 1) | (kind == 5), torch.randint(2, 200, (rows,), generator=g, device="cuda"), 0).to(torch.int32)
        x["top_p"] = torch.where((kind == 2) | (kind == 5), uniform((rows,), 0.5, 0.99), 1.0)
        x["min_p"] = torch.where((kind == 3) | (kind == 5), uniform((rows,), 0.01, 0.1), 0.0)
        x["temperature"] = torch.where(kind == 4, 0.0, x["temperature"])  # (greedy rows among the others)
    return x


# --------------------------------------------------------------------------------------------------- the plugin's form


@functools.lru_cache(maxsize=1)
def _client():
    from ryft_amd import pjrt
    return pjrt.load_plugin().client({"visible_devices": [0]})


@functools.lru_cache(maxsize=64)
def _executable(program):
    from ryft_amd import pjrt
    return _client().compile(pjrt.Program.mlir(program))


def _program(c, x):
    from ryft_amd import operators
    if c["family"] == "append":
        return operators.rope_append_module(
            tokens=c["tokens"], q_heads=c["hq"], kv_heads=c["hkv"], head_dim=c["d"], rotary_dim=c["rot"],
            pages=c["pages"], page_size=c["page"], dtype=c["dtype"], norm=c["norm"], eps=1e-6,
            interleaved=c["interleaved"])
    if c["family"] == "attention":
        return operators.paged_attention_module(
            tokens=x["q"].shape[0], sequences=c["sequences"], q_heads=c["hq"], kv_heads=c["hkv"], head_dim=c["d"],
            pages=x["k_cache"].shape[0], page_size=c["page"], pages_per_sequence=x["table"].shape[1], dtype=c["dtype"],
            scale=1.0 / math.sqrt(c["d"]), softcap=c["softcap"], window=c["window"], slopes=c["slopes"])
    return operators.sample_module(rows=c["rows"], vocab=c["vocab"], dtype=c["dtype"])


def prepare(case, seed):
    """The inputs, and the loaded executable that the plugin's form runs."""
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    if case["family"] == "attention":
        state["most"] = tuple(max(v) for v in _lengths(case))
    if own:
        state["exe"] = _executable(_program(case, x))
    torch.cuda.synchronize()
    return state


def _execute(exe, inputs, outputs):
    """The executable on torch's device memory and its current stream."""
    exe.execute_into([(t.data_ptr(), t.nbytes) for t in inputs], [(t.data_ptr(), t.nbytes) for t in outputs],
                     torch.cuda.current_stream().cuda_stream)
    return outputs


def _run_own(state):
    c, x, exe = state["case"], state["x"], state["exe"]
    if c["family"] == "append":
        ins = [x[n] for n in ("q", "k", "v", "positions", "slots", "freq", "k_cache", "v_cache")]
        if c["norm"]:
            ins += [x["q_weight"], x["k_weight"]]
        return _execute(exe, ins, [torch.empty_like(x["q"]), x["k_cache"], x["v_cache"]])
    if c["family"] == "attention":
        ins = [x[n] for n in ("q", "k_cache", "v_cache", "table", "starts", "lengths")]
        return _execute(exe, ins + ([x["slopes"]] if c["slopes"] else []), [torch.empty_like(x["q"])])
    rows, dev = c["rows"], x["logits"].device
    return _execute(exe, [x[n] for n in ("logits", "temperature", "top_k", "top_p", "min_p", "uniform")],
                    [torch.empty(rows, dtype=torch.int32, device=dev), torch.empty(rows, dtype=torch.float32, device=dev)])


# --------------------------------------------------------------------------------------------------- the plain form


def _rotated(c, x, cos, sin, weight):
    """Heads x[t, h, d] in 32 bits, normalised where there is a weight, their first `rot` values rotated."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6) * weight.float()
    rot = c["rot"]
    head, tail = x[..., :rot], x[..., rot:]
    if c["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((head, tail), dim=-1)


def _append_plain(c, x):
    angle = x["positions"].double()[:, None] * x["freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    dt = x["q"].dtype
    q = _rotated(c, x["q"], cos, sin, x.get("q_weight")).to(dt)
    k = _rotated(c, x["k"], cos, sin, x.get("k_weight")).to(dt)
    slot = x["slots"].long()
    page, at = slot // c["page"], slot % c["page"]
    x["k_cache"][page, :, at] = k
    x["v_cache"][page, :, at] = x["v"]
    return [q, x["k_cache"], x["v_cache"]]


def _attention_plain(c, x, most):
    """Every sequence padded to the longest: its queries and its keys gathered, and one batched softmax over them."""
    n, length = most
    b, hkv, d = c["sequences"], c["hkv"], c["d"]
    group, q, dev = c["hq"] // hkv, x["q"], x["q"].device
    starts, lengths = x["starts"].long(), x["lengths"].long()
    new = starts[1:] - starts[:-1]
    i, pos = torch.arange(n, device=dev), torch.arange(length, device=dev)
    token = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qs = q.float()[token].reshape(b, n, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * n, d)
    page = x["table"].long()[:, pos // c["page"]].clamp(min=0)
    at = (pos % c["page"]).expand(b, length)
    ks = x["k_cache"][page, :, at].float().permute(0, 2, 3, 1).contiguous()
    vs = x["v_cache"][page, :, at].float().permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(qs, ks).reshape(b, hkv, group, n, length) * (1.0 / math.sqrt(d))
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    where = (lengths - new)[:, None] + i                                    # position of each query
    away = pos[None, None] - where[:, :, None]                              # of each key from each query
    if c["slopes"]:
        s = s + x["slopes"].reshape(1, hkv, group, 1, 1) * away[:, None, None].float()
    seen = (away <= 0) & (pos < lengths[:, None, None]) & (i < new[:, None])[:, :, None]
    if c["window"]:
        seen = seen & (away > -c["window"])
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    o = torch.matmul(p.reshape(b, hkv, group * n, length), vs)
    o = o / p.sum(dim=-1).reshape(b, hkv, group * n, 1).clamp(min=1e-30)
    o = o.reshape(b, hkv, group, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, c["hq"], d)
    row = torch.searchsorted(starts, torch.arange(q.shape[0], device=dev), right=True) - 1
    return [o[row, torch.arange(q.shape[0], device=dev) - starts[row]].to(q.dtype)]


def _sample_plain(c, x):
    v = x["logits"].double()
    top = v.amax(dim=1, keepdim=True)
    greedy = x["temperature"].double()[:, None] == 0
    t = torch.where(greedy, 1.0, x["temperature"].double()[:, None])
    w = torch.exp((v - top) / t)
    order = torch.sort(v, dim=1, descending=True, stable=True).indices        # (equal logits: the lower index first)
    ws = w.gather(1, order)
    rank = torch.arange(c["vocab"], device=v.device)
    most = torch.where(x["top_k"] > 0, x["top_k"], c["vocab"]).long()[:, None]
    keep = (rank < torch.where(greedy, 1, most)) & (ws >= x["min_p"].double()[:, None])
    ws = ws * keep
    before = ws.cumsum(dim=1) - ws
    p = x["top_p"].double()[:, None]
    keep = keep & ((before < p * ws.sum(dim=1, keepdim=True)) | (p >= 1))
    w = w * torch.zeros_like(keep).scatter(1, order, keep)                    # the kept weights, by index again
    cum = w.cumsum(dim=1)
    total = cum[:, -1:]
    token = (cum <= x["uniform"].double()[:, None] * total).sum(dim=1, keepdim=True).clamp(max=c["vocab"] - 1)
    return [token[:, 0].to(torch.int32), torch.log(w.gather(1, token) / total)[:, 0].float()]


def run(state):
    if own:
        return _run_own(state)
    c, x = state["case"], state["x"]
    if c["family"] == "append":
        return _append_plain(c, x)
    if c["family"] == "attention":
        return _attention_plain(c, x, state["most"])
    return _sample_plain(c, x)


# --------------------------------------------------------------------------------------------------- measures


def work(case):
    c = case
    if c["family"] == "append":
        t, d, es = c["tokens"], c["d"], _DTYPE[c["dtype"]].itemsize
        values = t * (c["hq"] + 2 * c["hkv"]) * d
        return {"flops": 4.0 * t * (c["hq"] + c["hkv"]) * (c["rot"] + (d if c["norm"] else 0)),
                "bytes": 2 * es * values + 8 * t + 2 * c["rot"] + (2 * es * d if c["norm"] else 0)}
    if c["family"] == "attention":
        es, d, pairs, keys = _DTYPE[c["dtype"]].itemsize, c["d"], 0, 0
        new, total = _lengths(c)
        for n, length in zip(new, total):
            window = c["window"] or length
            first = max(0, length - n + 1 - window)                           # the first key that a query sees
            keys += length - first
            pairs += sum(min(window, length - n + i + 1) for i in range(n))
        return {"flops": 4.0 * c["hq"] * d * pairs,
                "bytes": 2 * es * (keys * c["hkv"] * d + sum(new) * c["hq"] * d) + 4 * (keys // c["page"] + 2 * len(new))}
    return {"flops": 0.0, "bytes": c["rows"] * (c["vocab"] * _DTYPE[c["dtype"]].itemsize + 28)}


def _exact_append(c, x):
    rot = c["rot"]

    def turned(t, weight):
        t = t.double()
        if weight is not None:
            t = t / torch.sqrt(t.square().mean(dim=-1, keepdim=True) + 1e-6) * weight.double()
        pairs = t[..., :rot].unflatten(-1, (rot // 2, 2)) if c["interleaved"] else t[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=t.device), x["positions"].double()[:, None, None] * x["freq"].double())
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        t = t.clone()
        t[..., :rot] = (pairs if c["interleaved"] else pairs.transpose(-1, -2)).flatten(-2)
        return t

    caches = []
    for cache, rows in ((x["k_cache"], turned(x["k"], x.get("k_weight"))), (x["v_cache"], x["v"].double())):
        flat = cache.double().transpose(1, 2).reshape(-1, c["hkv"], c["d"])   # one row for each slot
        flat[x["slots"].long()] = rows
        caches.append(flat.reshape(c["pages"], c["page"], c["hkv"], c["d"]).transpose(1, 2).contiguous())
    return [turned(x["q"], x.get("q_weight"))] + caches


def _exact_attention(c, x):
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    at, group = 0, c["hq"] // c["hkv"]
    for i, (n, length) in enumerate(zip(*_lengths(c))):
        pages = x["table"][i, :-(-length // c["page"])].long()
        k, v = (x[m][pages].double().transpose(1, 2).reshape(-1, c["hkv"], c["d"])[:length] for m in ("k_cache", "v_cache"))
        for first in range(0, n, 256):                                       # 256 queries of a sequence at a time
            last = min(n, first + 256)
            pos = torch.arange(length - n + first, length - n + last, device="cuda")[:, None]
            key = torch.arange(length, device="cuda")[None]
            hide = key > pos
            if c["window"]:
                hide |= pos - key >= c["window"]
            for h in range(c["hq"]):
                s = x["q"][at + first:at + last, h].double() @ k[:, h // group].t().contiguous() / math.sqrt(c["d"])
                if c["softcap"]:
                    s = torch.tanh(s / c["softcap"]) * c["softcap"]
                if c["slopes"]:
                    s = s - x["slopes"][h].double() * (pos - key)
                out[at + first:at + last, h] = torch.softmax(s.masked_fill(hide, float("-inf")), dim=-1) @ v[:, h // group]
        at += n
    return [out]


def _exact_sample(c, x):
    tokens, logs = [], []
    logits = x["logits"].double().cpu().numpy()
    t, k, p, m, u = (x[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
    for r in range(c["rows"]):
        row = logits[r]
        if t[r] == 0:
            tokens.append(int(np.argmax(row)))
            logs.append(0.0)
            continue
        w = np.exp((row - row.max()) / t[r])
        kept = np.lexsort((np.arange(row.size), -row))                        # by logit, then by index
        kept = kept[:int(k[r])] if k[r] > 0 else kept
        kept = kept[w[kept] >= m[r]]
        if p[r] < 1:
            mass = np.cumsum(w[kept])
            kept = kept[:1 + int(np.count_nonzero(mass[:-1] < p[r] * mass[-1]))]
        kept = np.sort(kept)
        mass = np.cumsum(w[kept])
        i = min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), kept.size - 1)
        tokens.append(int(kept[i]))
        logs.append(math.log(w[kept[i]] / mass[-1]))
    return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(logs, dtype=torch.float64)]


def exact(case, seed):
    x = _inputs(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["family"]](case, x)
