"""Timed operators of a step that verifies drafted tokens: attention of a tree of drafted tokens over a paged cache, the
products with 4-bit weights whose time such steps are, and the acceptance of the tree's longest matching path. Each has a
plain form of elementary torch operations (`own` false) and the plugin's form (`own` true): a module with the operator's
`stablehlo.custom_call`, compiled once, run on the caller's device memory and stream.

Families (`family` of a case):

* ``int4``    rows of activations against a weight of 4-bit integers with a scale (and a zero point) for each group of a
              row's values. Result: the products.
* ``tree``    queries of several sequences' drafted tokens against the pages of the cache: every committed token, and of
              the drafted ones those that a bit mask names (a token's ancestors and itself). Result: the outputs.
* ``accept``  the longest path of each tree along which the drafted tokens are those that the model chose. Results: how
              many tokens each sequence gets, which, the nodes they come from, and the caches with the path's keys and
              values moved to the positions behind the committed ones.
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
        # one token against a square projection: the smallest product, bounded by latency
        dict(name="int4_one", family="int4", rows=1, k=4096, n=4096, group=128, dtype="bf16", zeros=False),
        # a decoding step of 16 sequences against gate and up projections together
        dict(name="int4_step", family="int4", rows=16, k=4096, n=28672, group=128, dtype="bf16", zeros=True),
        # the trees of four sequences against a long down projection
        dict(name="int4_trees", family="int4", rows=256, k=14336, n=4096, group=64, dtype="f16", zeros=False),
        # a prompt of 2048 tokens
        dict(name="int4_prompt", family="int4", rows=2048, k=4096, n=12288, group=128, dtype="bf16", zeros=True),
        # odd numbers of rows and columns, small groups
        dict(name="int4_odd", family="int4", rows=33, k=2080, n=7001, group=32, dtype="f16", zeros=True),
        # eight drafted tokens of one short sequence: the smallest call
        dict(name="tree_one", family="tree", sequences=1, nodes=8, context=500, ragged=False, hq=8, hkv=8, d=64,
             dtype="bf16", page=16, window=0, softcap=0.0),
        # trees of up to 64 tokens of 16 sequences of all lengths
        dict(name="tree_batch", family="tree", sequences=16, nodes=64, context=4096, ragged=True, hq=32, hkv=8, d=128,
             dtype="bf16", page=16, window=0, softcap=0.0),
        # two long sequences, capped scores: the key axis is all the parallelism there is
        dict(name="tree_long", family="tree", sequences=2, nodes=32, context=60000, ragged=False, hq=16, hkv=2, d=128,
             dtype="f16", page=32, window=0, softcap=30.0),
        # wide trees with a window
        dict(name="tree_wide", family="tree", sequences=4, nodes=256, context=12000, ragged=True, hq=16, hkv=4, d=64,
             dtype="bf16", page=64, window=4096, softcap=0.0),
        # one tree, one layer's caches: the smallest call
        dict(name="accept_one", family="accept", sequences=1, nodes=8, ragged=False, hkv=8, d=64, dtype="bf16", page=16,
             layers=1),
        # 64 trees, the caches of eight layers
        dict(name="accept_batch", family="accept", sequences=64, nodes=64, ragged=True, hkv=8, d=128, dtype="bf16",
             page=16, layers=8),
    ]


def _size(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; odd ones as likely as even ones."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.choice(["int4", "int4", "tree", "tree", "accept"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if family == "int4":
        while True:
            group = rng.choice([32, 64, 128, 128])
            rows, k, n = _size(rng, 1, 2048), group * _size(rng, 1024 // group, 16384 // group), _size(rng, 256, 32768)
            if rows * k * n <= 1 << 36:
                return dict(family="int4", rows=rows, k=k, n=n, group=group, dtype=dtype, zeros=rng.random() < 0.5)
    hkv, d, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if family == "tree":
        group = rng.choice([1, 2, 4, 5, 8])
        while True:
            b, nodes, context = _size(rng, 1, 64), _size(rng, 2, 256), _size(rng, 16, 65536)
            if b * hkv * group * nodes * (context + nodes) <= 1 << 27 and b * (context + nodes) * hkv * d <= 1 << 26:
                return dict(family="tree", sequences=b, nodes=nodes, context=context, ragged=rng.random() < 0.7,
                            hq=hkv * group, hkv=hkv, d=d, dtype=dtype, page=page,
                            window=rng.choice([0, 0, _size(rng, 512, 8192)]), softcap=rng.choice([0.0, 0.0, 30.0, 50.0]))
    while True:
        b, nodes, layers = _size(rng, 1, 256), _size(rng, 2, 256), rng.randint(1, 16)
        if b * nodes * hkv * d * layers <= 1 << 25:
            return dict(family="accept", sequences=b, nodes=nodes, ragged=rng.random() < 0.7, hkv=hkv, d=d, dtype=dtype,
                        page=page, layers=layers)


_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _lengths(c):
    """Drafted tokens and committed tokens of each sequence: spread evenly where they differ."""
    nodes, prior = [], []
    for i in range(c["sequences"]):
        f, g = ((i + 1) * 0.6180339887) % 1.0, ((i + 1) * 0.7548776662) % 1.0
        nodes.append(max(1, math.ceil(c["nodes"] * (0.25 + 0.75 * f))) if c["ragged"] else c["nodes"])
        prior.append(int(c.get("context", 0) * g) if c["ragged"] else c.get("context", 0))
    return nodes, prior


def _trees(nodes, seed):
    """A random tree for each sequence: each node's parent (-1: the root, which is the last committed choice), and the
    bits of its ancestors and itself in words of 32."""
    r = np.random.RandomState(seed % (1 << 32))
    words = -(-max(nodes) // 32)
    parents, masks = [], []
    for n in nodes:
        up = [-1] + [int(r.randint(0, j)) for j in range(1, n)]
        seen = []
        for j, p in enumerate(up):
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
        parents += up
        masks += [s.to_bytes(4 * words, "little") for s in seen]
    return np.array(parents, dtype=np.int32), np.frombuffer(b"".join(masks), dtype="<i4").reshape(-1, words).copy()


def _choices(nodes, parents, seed):
    """Drafted tokens and the model's choice after each node, along a random path from each root down as the drafts say.
    The path's nodes stand in their own places or behind all places that the path fills, so that a call repeated on its
    own results gives the same again."""
    r = np.random.RandomState((seed + 1) % (1 << 32))
    tokens, targets = r.randint(0, 32000, parents.size).astype(np.int32), r.randint(32000, 64000, parents.size).astype(np.int32)
    at = 0
    for n in nodes:
        children = [[] for _ in range(n)]
        for j in range(1, n):
            children[parents[at + j]].append(j)
        path = [0]
        while children[path[-1]] and r.rand() < 0.85:
            longer = path + [children[path[-1]][r.randint(len(children[path[-1]]))]]
            if any(p != i and p < len(longer) for i, p in enumerate(longer)):
                break
            path = longer
        for a, b in zip(path, path[1:]):
            for j in children[a]:
                if j < b and tokens[at + j] == tokens[at + b]:                # (the lowest of equal children is taken)
                    tokens[at + j] = 64000
            targets[at + a] = tokens[at + b]
        at += n
    return tokens, targets


# --------------------------------------------------------------------------------------------------- inputs


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPE[c["dtype"]]

    def normal(shape, std=1.0, dtype=None):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype or dt)

    def whole(lo, hi, shape, dtype):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=dtype)

    if c["family"] == "int4":
        groups = c["k"] // c["group"]
        x = {"x": normal((c["rows"], c["k"])), "weight": whole(0, 256, (c["n"], c["k"] // 2), torch.uint8),
             "scale": torch.rand((c["n"], groups), generator=g, device="cuda").mul_(0.01).add_(0.002).to(dt)}
        if c["zeros"]:
            x["zero"] = whole(5, 12, (c["n"], groups), torch.uint8)
        return x
    nodes, prior = _lengths(c)
    page, d = c["page"], c["d"]
    parents, visible = _trees(nodes, int(seed))
    x = {"starts": torch.tensor(np.cumsum([0] + nodes), dtype=torch.int32).cuda(), "visible": torch.from_numpy(visible).cuda()}
    if c["family"] == "tree":
        total = [n + p for n, p in zip(nodes, prior)]
        need = [-(-n // page) for n in total]
        pages = sum(need) + 7
        order = torch.randperm(pages, generator=g, device="cuda").cpu()  # (pages are handed out in no order)
        table, at = torch.full((c["sequences"], -(-(c["context"] + c["nodes"]) // page)), -1, dtype=torch.int32), 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        cache = (pages, c["hkv"], page, d)
        x.update(q=normal((sum(nodes), c["hq"], d), 1.5), k_cache=normal(cache), v_cache=normal(cache), table=table.cuda(),
                 lengths=torch.tensor(total, dtype=torch.int32).cuda())
        return x
    tokens, targets = _choices(nodes, parents, int(seed))
    pages = -(-sum(nodes) // page) + 5
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:sum(nodes)].to(torch.int32)
    x.update(tokens=torch.from_numpy(tokens).cuda(), parents=torch.from_numpy(parents).cuda(),
             targets=torch.from_numpy(targets).cuda(), slots=slots,
             caches=[normal((pages, c["hkv"], page, d)) for _ in range(2 * c["layers"])])
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
    if c["family"] == "int4":
        return operators.int4_matmul_module(rows=c["rows"], inner=c["k"], columns=c["n"], group=c["group"],
                                            dtype=c["dtype"], zeros=c["zeros"])
    if c["family"] == "tree":
        return operators.tree_attention_module(
            tokens=x["q"].shape[0], sequences=c["sequences"], q_heads=c["hq"], kv_heads=c["hkv"], head_dim=c["d"],
            pages=x["k_cache"].shape[0], page_size=c["page"], pages_per_sequence=x["table"].shape[1],
            words=x["visible"].shape[1], dtype=c["dtype"], scale=1.0 / math.sqrt(c["d"]), softcap=c["softcap"],
            window=c["window"])
    return operators.tree_accept_module(
        tokens=x["tokens"].shape[0], sequences=c["sequences"], caches=2 * c["layers"], pages=x["caches"][0].shape[0],
        kv_heads=c["hkv"], page_size=c["page"], head_dim=c["d"], dtype=c["dtype"])


def prepare(case, seed):
    """The inputs, and the loaded executable that the plugin's form runs."""
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    if case["family"] != "int4":
        nodes, prior = _lengths(case)
        state["most"] = max(nodes), max(prior)
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
    if c["family"] == "int4":
        ins = [x[n] for n in ("x", "weight", "scale")] + ([x["zero"]] if c["zeros"] else [])
        return _execute(exe, ins, [torch.empty((c["rows"], c["n"]), dtype=x["x"].dtype, device=x["x"].device)])
    if c["family"] == "tree":
        ins = [x[n] for n in ("q", "k_cache", "v_cache", "table", "starts", "lengths", "visible")]
        return _execute(exe, ins, [torch.empty_like(x["q"])])
    ins = [x[n] for n in ("tokens", "parents", "targets", "slots", "starts")]
    outs = [torch.empty(c["sequences"], dtype=torch.int32, device="cuda"), torch.empty_like(x["tokens"]), torch.empty_like(x["tokens"])]
    return _execute(exe, ins + x["caches"], outs + x["caches"])


# --------------------------------------------------------------------------------------------------- the plain form


def _int4_plain(c, x):
    w = x["weight"]
    q = torch.stack((w & 15, w >> 4), dim=-1).float().reshape(c["n"], -1, c["group"])
    q = q - (x["zero"].float().unsqueeze(-1) if c["zeros"] else 8.0)
    w = (q * x["scale"].float().unsqueeze(-1)).reshape(c["n"], c["k"])
    return [torch.matmul(x["x"].float(), w.t()).to(x["x"].dtype)]


def _sequence_of(starts, tokens):
    """The sequence of each row, and its place in it."""
    row = torch.arange(tokens, device=starts.device)
    b = torch.searchsorted(starts, row, right=True) - 1
    return b, row - starts[b]


def _bits(visible):
    """visible's bits as truth values [rows, 32 · words]."""
    shift = torch.arange(32, device=visible.device, dtype=torch.int32)
    return ((visible.unsqueeze(-1) >> shift) & 1).flatten(1) != 0


def _tree_plain(c, x, most):
    """Every sequence padded to the longest: its queries and its keys gathered, and one batched softmax over them."""
    n, prior = most
    b, hkv, d = c["sequences"], c["hkv"], c["d"]
    length = n + prior
    group, q, dev = c["hq"] // hkv, x["q"], x["q"].device
    starts, lengths = x["starts"].long(), x["lengths"].long()
    new = starts[1:] - starts[:-1]
    first = lengths - new                                                   # position of the first drafted token
    i, pos = torch.arange(n, device=dev), torch.arange(length, device=dev)
    token = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qs = q.float()[token].reshape(b, n, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * n, d)
    page = x["table"].long()[:, (pos // c["page"]).clamp(max=x["table"].shape[1] - 1)].clamp(min=0)
    at = (pos % c["page"]).expand(b, length)
    ks = x["k_cache"][page, :, at].float().permute(0, 2, 3, 1).contiguous()
    vs = x["v_cache"][page, :, at].float().permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(qs, ks).reshape(b, hkv, group, n, length) * (1.0 / math.sqrt(d))
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    bits = _bits(x["visible"])[token]                                       # [b, n, 32 · words]
    node = pos - first[:, None]                                             # of each key, negative for committed ones
    drafted = bits.gather(2, node.clamp(min=0, max=bits.shape[2] - 1)[:, None].expand(b, n, length))
    inside = (node < new[:, None])[:, None]
    seen = torch.where((node < 0)[:, None], True, drafted & inside)
    if c["window"]:
        where = first[:, None] + bits.sum(dim=2) - 1                        # a query's position: its depth in the tree
        seen = seen & ((node >= 0)[:, None] | (where[:, :, None] - pos < c["window"]))
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    o = torch.matmul(p.reshape(b, hkv, group * n, length), vs)
    o = o / p.sum(dim=-1).reshape(b, hkv, group * n, 1).clamp(min=1e-30)
    o = o.reshape(b, hkv, group, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, c["hq"], d)
    row, place = _sequence_of(starts, q.shape[0])
    return [o[row, place].to(q.dtype)]


def _accept_plain(c, x):
    """A node is on the path if it and all its ancestors are the lowest child that their parent's choice names."""
    tokens, targets, starts = x["tokens"], x["targets"], x["starts"].long()
    count, dev = tokens.shape[0], tokens.device
    row, place = _sequence_of(starts, count)
    up = x["parents"].long()
    child = (up >= 0) & (up < place)
    parent = torch.where(child, starts[row] + up, 0)
    child = child & (tokens == targets[parent])
    rows = torch.arange(count, device=dev)
    low = torch.full((count + 1,), count, device=dev).scatter_reduce(0, torch.where(child, parent, count), rows, "amin")
    chosen = (place == 0) | (child & (low[parent] == rows))
    bits = _bits(x["visible"])
    node = torch.arange(bits.shape[1], device=dev)
    on = (~bits | chosen[(starts[row][:, None] + node).clamp(max=count - 1)]).all(dim=1)
    at = torch.where(on, starts[row] + bits.sum(dim=1) - 1, count)           # the place that a node of the path fills
    path = torch.full((count + 1,), -1, dtype=torch.int32, device=dev).scatter(0, at, place.to(torch.int32))[:count]
    source = torch.where(path >= 0, starts[row] + path, rows)
    emitted = torch.where(path >= 0, targets[source], -1)
    counts = torch.zeros(c["sequences"], dtype=torch.int32, device=dev).scatter_add(0, row, on.to(torch.int32))
    slot = x["slots"].long()
    src, dst, page = slot[source], slot, c["page"]
    for cache in x["caches"]:
        cache[dst // page, :, dst % page] = cache[src // page, :, src % page]
    return [counts, emitted, path] + x["caches"]


def run(state):
    if own:
        return _run_own(state)
    c, x = state["case"], state["x"]
    if c["family"] == "int4":
        return _int4_plain(c, x)
    if c["family"] == "tree":
        return _tree_plain(c, x, state["most"])
    return _accept_plain(c, x)


# --------------------------------------------------------------------------------------------------- measures


def work(case):
    c, es = case, _DTYPE[case["dtype"]].itemsize
    if c["family"] == "int4":
        t, k, n, groups = c["rows"], c["k"], c["n"], c["k"] // c["group"]
        return {"flops": 2.0 * t * k * n, "bytes": n * k // 2 + n * groups * (es + c["zeros"]) + es * t * (k + n)}
    nodes, prior = _lengths(c)
    words = -(-max(nodes) // 32)
    if c["family"] == "tree":
        d, keys, pairs = c["d"], 0, 0
        for n, p in zip(nodes, prior):
            keys += n + min(p, c["window"] or p)
            pairs += n * (min(p, c["window"] or p) + math.ceil(math.log2(n + 1)))  # (about as many ancestors)
        return {"flops": 4.0 * c["hq"] * d * pairs,
                "bytes": 2 * es * (keys * c["hkv"] * d + sum(nodes) * c["hq"] * d) + 4 * (keys // c["page"] + sum(nodes) * words)}
    # (of each sequence about one node moves, read and written in every cache)
    return {"flops": 0.0, "bytes": 24 * sum(nodes) + 2 * 2 * c["layers"] * c["sequences"] * c["hkv"] * c["d"] * es}


def _exact_int4(c, x):
    rows = []
    for lo in range(0, c["n"], 2048):                                        # 2048 columns of the result at a time
        w = x["weight"][lo:lo + 2048].to(torch.int64)
        q = torch.empty((w.shape[0], c["k"]), dtype=torch.float64, device=w.device)
        q[:, 0::2], q[:, 1::2] = (w % 16).double(), (w // 16).double()
        per = torch.arange(c["k"], device=w.device) // c["group"]
        zero = x["zero"][lo:lo + 2048].double()[:, per] if c["zeros"] else 8.0
        rows.append(x["x"].double() @ ((q - zero) * x["scale"][lo:lo + 2048].double()[:, per]).t().contiguous())
    return [torch.cat(rows, dim=1)]


def _exact_tree(c, x):
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    visible = x["visible"].cpu().numpy().view(np.uint32)
    at, group = 0, c["hq"] // c["hkv"]
    for i, (n, prior) in enumerate(zip(*_lengths(c))):
        length = n + prior
        pages = x["table"][i, :-(-length // c["page"])].long()
        k, v = (x[m][pages].double().transpose(1, 2).reshape(-1, c["hkv"], c["d"])[:length] for m in ("k_cache", "v_cache"))
        hide = np.zeros((n, length), dtype=bool)
        for j in range(n):
            mine = [a for a in range(n) if visible[at + j, a // 32] >> np.uint32(a % 32) & 1]
            hide[j, prior:] = True
            hide[j, [prior + a for a in mine]] = False
            if c["window"]:
                hide[j, :max(0, min(prior, prior + len(mine) - c["window"]))] = True
        hide = torch.from_numpy(hide).cuda()
        for h in range(c["hq"]):
            s = x["q"][at:at + n, h].double() @ k[:, h // group].t().contiguous() / math.sqrt(c["d"])
            if c["softcap"]:
                s = torch.tanh(s / c["softcap"]) * c["softcap"]
            out[at:at + n, h] = torch.softmax(s.masked_fill(hide, float("-inf")), dim=-1) @ v[:, h // group]
        at += n
    return [out]


def _exact_accept(c, x):
    tokens, parents, targets, slots = (x[n].cpu().numpy() for n in ("tokens", "parents", "targets", "slots"))
    counts, emitted, path = [], np.full(tokens.size, -1, dtype=np.int32), np.full(tokens.size, -1, dtype=np.int32)
    at, moves = 0, []
    for n in _lengths(c)[0]:
        here, walked = 0, [0]
        while True:
            below = [j for j in range(here + 1, n) if parents[at + j] == here and tokens[at + j] == targets[at + here]]
            if not below:
                break
            here = below[0]
            walked.append(here)
        counts.append(len(walked))
        for j, node in enumerate(walked):
            emitted[at + j], path[at + j] = targets[at + node], node
            moves.append((slots[at + node], slots[at + j]))
        at += n
    src, dst = (torch.tensor([m[e] for m in moves], device="cuda").long() for e in (0, 1))
    caches = []
    for cache in x["caches"]:
        flat = cache.double().transpose(1, 2).reshape(-1, c["hkv"], c["d"])   # one row for each slot
        flat[dst] = flat[src].clone()
        caches.append(flat.reshape(cache.shape[0], c["page"], c["hkv"], c["d"]).transpose(1, 2).contiguous())
    return [torch.tensor(counts, dtype=torch.int32), torch.from_numpy(emitted), torch.from_numpy(path)] + caches


def exact(case, seed):
    x = _inputs(case, seed)
    return {"int4": _exact_int4, "tree": _exact_tree, "accept": _exact_accept}[case["family"]](case, x)
