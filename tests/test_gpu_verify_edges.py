"""The operators that verify drafted tokens on the GPU at the ends of what their definitions allow: infinities, sums that
leave f32's range on the way, calls without tokens, starts that are no starts.

int4_matmul's sums carry a bias of 16 beside each value, so that an infinity of x, or a large finite one, can make them
infinite or NaN where the definition is not; such results are summed again in 64 bits. Where the definition is infinite or
NaN the results are that exactly. Finite results: `int4_error` and half a step of the type, as in test_gpu_verify.py; results
summed again are nearer (64 bits, rounded to f32 and to the type)."""
import numpy as np
import pytest
import torch  # (before the plugin: both then use one HIP runtime)

from oracle import operators as oo
from oracle import stablehlo as sh
from ryft_amd import operators, pjrt
from tests import operator_programs as op
from tests import verify_programs as vp
from tests.test_gpu_operators import attention_error, close, run

pytestmark = pytest.mark.gpu

# one of each way through the kernels: rows through the ring and in registers, with more tiles than workgroups, tiles in one
# range of K and in several, results of a number that is no multiple of four, and the kernel for any type and group
PATHS = {
    "one": (1, 512, 40, 128, "bf16"),
    "ring": (5, 4096, 70, 64, "f16"),
    "registers": (16, 512, 4100, 32, "bf16"),
    "registers_4": (3, 8192, 4200, 128, "bf16"),
    "more_tiles": (2, 256, 8230, 64, "bf16"),
    "tile": (70, 256, 300, 128, "bf16"),
    "tile_f16": (70, 256, 301, 32, "f16"),
    "tiles_of_128": (300, 160, 3000, 32, "bf16"),
    "parts": (40, 4096, 257, 128, "bf16"),
    "parts_odd": (33, 2080, 71, 32, "f16"),
    "other_groups": (20, 480, 33, 48, "bf16"),
    "f32": (20, 512, 33, 64, "f32"),
}


def definition(x):
    with np.errstate(invalid="ignore", over="ignore"):
        return oo.int4_matmul(x, {})[0]


@pytest.mark.parametrize("zeros", [False, True], ids=["eight", "zeros"])
@pytest.mark.parametrize("out", ["f32", "same"])
@pytest.mark.parametrize("name", PATHS)
def test_int4_matmul_of_infinities(gpu_client, name, out, zeros):
    # an infinity is ±inf by the sign of its weight, NaN where that is zero or another infinity has the other sign
    rows, inner, columns, group, dtype = PATHS[name]
    out = dtype if out == "same" else out
    module, ins = vp.int4_case(rows, inner, columns, group, dtype, zeros=zeros, out_dtype=out, seed=rows + inner)
    x = vp.values(ins)
    x[0][0, 7] = np.inf
    if rows > 1:
        x[0][rows - 1, inner - 1] = -np.inf
    if rows > 2:
        x[0][1, 3], x[0][1, inner - 2] = np.inf, -np.inf
    if rows > 4:
        x[0][2, inner // 2], x[0][3, 0], x[0][3, 1] = np.nan, np.inf, np.nan
    if rows > 16:
        x[0][16:rows:9, inner // 3] = np.inf
    ins[0] = op.host(x[0], dtype)
    (got,), _ = run(gpu_client, module, ins, [out])
    want = definition(vp.values(ins))
    odd = ~np.isfinite(x[0]).all(axis=1)
    assert np.isinf(want[0]).any() and (np.isnan(want[0]).any() or columns < 50)
    assert np.array_equal(got[odd], want[odd], equal_nan=True)
    close(got[~odd], want[~odd], out, vp.int4_error([x[0][~odd], *x[1:]]) + 2.0 ** -25, "others")


@pytest.mark.parametrize("power", [108, 114, 120, 125])
@pytest.mark.parametrize("name", [n for n in PATHS if PATHS[n][4] != "f16"])
def test_int4_matmul_of_the_largest_values(gpu_client, name, power):
    # zero points up to 255 and values up to 2^127: sums of (16 + z) x pass f32's range, results are around 2^(power - 20)
    rows, inner, columns, group, dtype = PATHS[name]
    module, ins = vp.int4_case(rows, inner, columns, group, dtype, zeros=True, scale_dtype="f32", out_dtype="f32", seed=power + rows)
    r = np.random.RandomState(power)
    ins[0] = op.host(r.uniform(-3.9, 3.9, (rows, inner)) * 2.0 ** power, dtype)
    ins[2] = op.host(r.uniform(0.5, 1, ins[2].dims) * 2.0 ** -35, "f32")
    ins[3] = vp.host(r.randint(0, 256, ins[3].dims), "ui8")
    (got,), _ = run(gpu_client, module, ins, ["f32"])
    x = vp.values(ins)
    want = definition(x)
    assert np.isfinite(want.astype(np.float32)).all()
    close(got, want, "f32", vp.int4_error(x), "y")


@pytest.mark.parametrize("name", [n for n in PATHS if PATHS[n][4] != "f16"])
def test_int4_matmul_of_sums_that_come_back(gpu_client, name):
    # the second half of a row takes off what the first has put beyond f32's largest value: what is left is one value of x, a
    # power of two, times the column's number, exactly
    rows, inner, columns, group, dtype = PATHS[name]
    half = inner // 2 // group * group
    module, ins = vp.int4_case(rows, inner, columns, group, dtype, out_dtype="f32", scale_dtype="f32", seed=2)
    x, q = np.zeros((rows, inner)), np.full((columns, inner), 8)
    x[:, :half] = 2.0 ** 127
    x[:, half:2 * half] = -2.0 ** 127
    x[:, half] = -2.0 ** 120
    q[:, :2 * half] = 11
    q[:, 0], q[:, half] = 8, 8 + np.arange(columns) % 8
    ins[0] = op.host(x, dtype)
    ins[1] = vp.host(q[:, 0::2] | q[:, 1::2] << 4, "ui8")
    ins[2] = op.host(np.ones(ins[2].dims), "f32")
    (got,), _ = run(gpu_client, module, ins, ["f32"])
    assert np.array_equal(got, np.broadcast_to(-2.0 ** 120 * (np.arange(columns) % 8), got.shape))


@pytest.mark.parametrize("name", PATHS)
def test_int4_matmul_of_scales_that_are_not_finite(gpu_client, name):
    rows, inner, columns, group, dtype = PATHS[name]
    module, ins = vp.int4_case(rows, inner, columns, group, dtype, scale_dtype="f32", out_dtype="f32", seed=9)
    x = vp.values(ins)
    groups = inner // group
    x[2][3, groups - 1], x[2][columns - 1, 0], x[2][20, groups // 2] = np.nan, np.inf, -np.inf
    ins[2] = op.host(x[2], "f32")
    (got,), _ = run(gpu_client, module, ins, ["f32"])
    want = definition(x)
    odd = ~np.isfinite(x[2]).all(axis=1)
    assert odd.sum() == 3 and np.array_equal(got[:, odd], want[:, odd], equal_nan=True)
    close(got[:, ~odd], want[:, ~odd], "f32", vp.int4_error([x[0], x[1][~odd], x[2][~odd]]), "others")


@pytest.mark.parametrize("rows, inner, columns, group", [(1400, 13248, 6144, 64), (300, 32768, 70, 128), (40, 1 << 20, 20, 128)], ids=str)
def test_int4_matmul_of_infinities_in_later_goes(gpu_client, rows, inner, columns, group):
    # rows that are prepared, or multiplied, in several goes: results that are summed again are those of their own rows
    module, ins = vp.int4_case(rows, inner, columns, group, "bf16", zeros=True, out_dtype="f32", seed=rows)
    raw = np.array(ins[0].data).reshape(rows, inner)
    some = [0, rows // 2 - 1, rows // 2, rows - 2, rows - 1]
    for n, t in enumerate(some[1:4]):
        raw[t, 11 * n], raw[t, inner - 1 - n] = (0x7F80, 0xFF80, 0x7FC0)[n], 0x7F80  # (inf, -inf, NaN; inf)
    ins[0] = type(ins[0])(raw, ins[0].type, ins[0].dims)
    given = [torch.from_numpy(np.array(i.data).view(np.int16 if i.data.dtype == np.uint16 else i.data.dtype)).cuda() for i in ins]
    y = torch.full((rows, columns), 7.0, device="cuda")
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    exe.execute_into([(g.data_ptr(), g.nbytes) for g in given], [(y.data_ptr(), y.nbytes)], torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = y[some].double().cpu().numpy()
    x = [sh.from_raw(raw[some], "bf16")] + vp.values(ins[1:])
    want = definition(x)
    assert np.array_equal(got[1:4], want[1:4], equal_nan=True) and not np.isfinite(want[1:4]).any()
    close(got[[0, 4]], want[[0, 4]], "f32", vp.int4_error([x[0][[0, 4]], *x[1:]]), "others")
    assert int((~torch.isfinite(y)).any(dim=1).sum()) == 3


@pytest.mark.parametrize("name", ["one", "registers", "tile", "parts", "f32"])
def test_int4_matmul_of_infinities_in_a_replayed_graph(gpu_client, name):
    # the inputs change between replays: finite, with infinities and NaN, and finite again
    rows, inner, columns, group, dtype = PATHS[name]
    module, ins = vp.int4_case(rows, inner, columns, group, dtype, out_dtype="f32", seed=4)
    given = [torch.from_numpy(np.array(i.data).view(np.int16 if i.data.dtype == np.uint16 else i.data.dtype)).cuda() for i in ins]
    y = torch.full((rows, columns), 7.0, device="cuda")
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        exe.execute_into([(g.data_ptr(), g.nbytes) for g in given], [(y.data_ptr(), y.nbytes)], torch.cuda.current_stream().cuda_stream)
    x = vp.values(ins)
    odd = x[0].copy()
    odd[rows - 1, 5], odd[0, inner - 1] = np.inf, -np.inf
    if rows > 2:
        odd[1, 9] = np.nan
    for now in (x[0], odd, x[0], odd):
        raw = op.host(now, dtype)
        given[0].copy_(torch.from_numpy(np.array(raw.data).view(np.int16) if dtype != "f32" else np.array(raw.data)).reshape(given[0].shape))
        graph.replay()
        torch.cuda.synchronize()
        got, want = y.double().cpu().numpy(), definition([now, *x[1:]])
        some = np.isfinite(now).all(axis=1)
        assert np.array_equal(got[~some], want[~some], equal_nan=True)
        close(got[some], want[some], "f32", vp.int4_error([now[some], *x[1:]]), name)


@pytest.mark.parametrize("rows, inner, columns, group, dtype", [(250_001, 64, 33, 32, "bf16"), (110_000, 32, 300, 32, "f16"), (70_003, 2, 5, 2, "f32"),
                                                                (600_000, 48, 3, 48, "bf16")], ids=str)
def test_int4_matmul_of_many_rows(gpu_client, rows, inner, columns, group, dtype):
    # in several goes, and past the number of workgroups that one axis of a grid has; as exact as whole numbers are
    module, ins = vp.int4_case(rows, inner, columns, group, dtype, zeros=True, out_dtype="f32", exact=True, seed=rows)
    (got,), _ = run(gpu_client, module, ins, ["f32"])
    assert np.array_equal(got, oo.int4_matmul(vp.values(ins), {})[0])


# ------------------------------------------------------------------------------------------------ no tokens
def empty_modules():
    tree = operators.tree_attention_module(tokens=0, sequences=3, q_heads=4, kv_heads=2, head_dim=64, pages=5, page_size=16,
                                           pages_per_sequence=4, words=2, scale=0.125)
    accept = operators.tree_accept_module(tokens=0, sequences=3, caches=2, pages=5, kv_heads=2, page_size=16, head_dim=64)
    int4 = operators.int4_matmul_module(rows=0, inner=64, columns=10, group=32)
    cache = ((5, 2, 16, 64), "bf16")
    words = lambda *shape: (shape, "i32")  # noqa: E731
    return {
        "tree_attention": (tree, [((0, 4, 64), "bf16"), cache, cache, words(3, 4), words(4), words(3), words(0, 2)],
                           [((0, 4, 64), "bf16")]),
        "tree_accept": (accept, [words(0)] * 4 + [words(4), cache, cache], [words(3), words(0), words(0), cache, cache]),
        "int4_matmul": (int4, [((0, 64), "bf16"), ((10, 32), "ui8"), ((10, 2), "bf16")], [((0, 10), "bf16")]),
    }


@pytest.mark.parametrize("into", [False, True], ids=["execute", "execute_into"])
@pytest.mark.parametrize("name", ["tree_attention", "tree_accept", "int4_matmul"])
def test_no_tokens(gpu_client, name, into):
    # a tensor of no elements has the address 0
    module, ins, outs = empty_modules()[name]
    kind = {"bf16": torch.bfloat16, "i32": torch.int32, "ui8": torch.uint8}
    given = [torch.ones(s, dtype=kind[t], device="cuda") if t == "bf16" else torch.zeros(s, dtype=kind[t], device="cuda") for s, t in ins]
    if not into:
        host = [vp.host(g.cpu().float().numpy(), t) for g, (_, t) in zip(given, ins)]
        got, _ = run(gpu_client, module, host, [t for _, t in outs])
    else:
        exe = gpu_client.compile(pjrt.Program.mlir(module))
        made = [torch.full(s, 7, dtype=kind[t], device="cuda") for s, t in outs]
        assert given[0].data_ptr() == 0
        exe.execute_into([(g.data_ptr(), g.nbytes) for g in given], [(m.data_ptr(), m.nbytes) for m in made],
                         torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        got = [m.cpu().float().numpy() for m in made]
    assert [g.shape for g in got] == [s for s, _ in outs]
    if name == "tree_accept":
        assert not got[0].any() and all((g == 1).all() for g in got[3:])


# ------------------------------------------------------------------------------------------------ starts that are no starts
def guarded(shape, dtype, value):
    """A tensor between 64 KiB that no one may write, and what checks that."""
    n = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
    room = -(-n // 256) * 256
    whole = torch.full((room + (1 << 17),), 0x5A, dtype=torch.uint8, device="cuda")
    inner = whole[1 << 16:(1 << 16) + n].view(dtype).reshape(shape)
    inner.copy_(value)
    return inner, lambda: bool((whole[:1 << 16] == 0x5A).all() and (whole[(1 << 16) + n:] == 0x5A).all())


BAD_STARTS = [
    ([-5, 30, 20, 60], True),                      # (0 to 30, none, 20 to 60: the last two share rows)
    ([60, 0, 60, 0], False), ([0, 20, 20, 60], False), ([-2 ** 31, -1, -1, -1], False), ([61, 70, 2 ** 31 - 1, 60], False),
    ([2 ** 31 - 1, 40, 40, 60], False), ([10, 20, 5, 2 ** 31 - 1], True),
]


@pytest.mark.parametrize("starts, shared", BAD_STARTS, ids=str)
@pytest.mark.parametrize("page, heads, dtype", [(16, (2, 64), "bf16"), (5, (3, 7), "bf16"), (16, (1, 4), "f32")], ids=str)
def test_tree_accept_of_any_starts(gpu_client, starts, shared, page, heads, dtype):
    """What the definition gives where no row is in two sequences. Rows in two are written by both: counts are still those of
    each sequence alone, the results are node numbers and targets of some sequence, or -1, and rows of no sequence are -1."""
    module, ins = vp.accept_case([20, 20, 20], 2, *heads, page, dtype, vocab=1, wide=True, seed=2, bad_slots=page == 5)
    ins[4] = op.host(starts, "i32")
    x = vp.values(ins)
    kind = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    words = lambda a: torch.from_numpy(np.asarray(a).astype(np.int32))  # noqa: E731
    given = [guarded(a.shape, torch.int32, words(a)) for a in x[:5]] + \
            [guarded(a.shape, kind, torch.from_numpy(a).to(kind)) for a in x[5:]]
    made = [guarded(s, torch.int32, torch.tensor(77)) for s in ((3,), (60,), (60,))] + [guarded(a.shape, kind, torch.tensor(0)) for a in x[5:]]
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    exe.execute_into([(g.data_ptr(), g.nbytes) for g, _ in given], [(m.data_ptr(), m.nbytes) for m, _ in made],
                     torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert all(whole() for _, whole in given + made)
    for (g, _), a in zip(given, x):                                    # (operands are as they were)
        assert np.array_equal(g.double().cpu().numpy(), a)
    counts, emitted, path, *caches = (m.double().cpu().numpy() for m, _ in made)
    want = oo.tree_accept(x, {})
    assert np.array_equal(counts, want[0])
    if not shared:
        for got, w in zip((emitted, path, *caches), want[1:]):
            assert np.array_equal(got, w)
        return
    clamped = np.clip(starts, 0, 60)
    inside = [b for b in range(3) if clamped[b] < clamped[b + 1]]
    rows = np.zeros(60, dtype=bool)
    for b in inside:
        rows[clamped[b]:clamped[b + 1]] = True
    alone = [oo.tree_accept([*x[:4], np.array([clamped[b], clamped[b + 1]])], {}) for b in inside]
    for got, k in ((emitted, 1), (path, 2)):
        assert (got[~rows] == -1).all()
        assert np.any([got == w[k] for w in alone] + [got == -1], axis=0).all()
    named = {int(s) for s in x[3][rows]}
    for got, before in zip(caches, x[5:]):
        for slot in range(before.shape[0] * page):
            if slot not in named:
                assert np.array_equal(got[slot // page, :, slot % page], before[slot // page, :, slot % page]), slot


@pytest.mark.parametrize("starts", [s for s, shared in BAD_STARTS if not shared], ids=str)
@pytest.mark.parametrize("tokens, heads, dtype", [(15, (4, 2, 64), "bf16"), (60, (4, 2, 128), "f16"), (60, (2, 2, 64), "f32")], ids=str)
def test_tree_attention_of_any_starts(gpu_client, starts, tokens, heads, dtype):
    # starts do not decrease; where they do, a row's heads have what its sequence's range gives, or zeros (15 tokens, with starts
    # of a quarter: the kernel for few rows, which gives zeros to all)
    n = tokens // 3
    module, ins = vp.tree_case([n, n, n], [300, 200, 90], *heads, 16, dtype, seed=4, masks="random", words=2)
    ins[4] = op.host([s if abs(s) > 60 else s * tokens // 60 for s in starts], "i32")
    (got,), _ = run(gpu_client, module, ins, [dtype])
    x = vp.values(ins)
    want, = oo.tree_attention(x, op.config_of(module))
    zeros = ~got.any(axis=2) & (np.diff(starts) < 0).any()
    close(got[~zeros], want[~zeros], dtype, attention_error(x, dtype), str(starts))
    assert not got[~want.any(axis=(1, 2))].any()


@pytest.mark.parametrize("nodes, heads, dtype", [([5, 3], (2, 2, 64), "bf16"), ([40, 70], (4, 2, 128), "f16"), ([20, 9], (2, 1, 64), "f32")],
                         ids=str)
def test_bits_past_the_last_node_stand_for_nothing(gpu_client, nodes, heads, dtype):
    # neither keys nor, under a window, a query's place in the text
    module, ins = vp.tree_case(nodes, [n + 200 for n in nodes], *heads, 16, dtype, words=4, window=60, seed=sum(nodes))
    (want,), _ = run(gpu_client, module, ins, [dtype])
    bits = vp.values(ins)[6]
    past = np.concatenate([np.broadcast_to([sum(1 << j for j in range(32) if 32 * w + j >= n) for w in range(4)], (n, 4)) for n in nodes])
    ins[6] = op.host((bits.astype(np.int64) & 0xffffffff | past).astype(np.uint32).view(np.int32), "i32")
    (got,), _ = run(gpu_client, module, ins, [dtype])
    assert (vp.values(ins)[6] != bits).any() and want.any() and np.array_equal(got, want)
    oracle, = oo.tree_attention(vp.values(ins), op.config_of(module))
    close(got, oracle, dtype, attention_error(vp.values(ins), dtype), "y")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("masks, window", [("tree", 0), ("tree", 40), ("random", 900)])
def test_tree_attention_of_large_trees(gpu_client, masks, window, dtype):
    # trees of many words, larger than the window, most of a sequence, or all of it
    nodes = [1100, 700, 33]
    module, ins = vp.tree_case(nodes, [1300, 700, 900], 2, 1, 64, 16, dtype, masks=masks, window=window, seed=window + 5)
    (got,), _ = run(gpu_client, module, ins, [dtype])
    x = vp.values(ins)
    want, = oo.tree_attention(x, op.config_of(module))
    close(got, want, dtype, attention_error(x, dtype), masks)
    assert not got[~want.any(axis=(1, 2))].any()


# ------------------------------------------------------------------------------------------------ the longest rows
@pytest.mark.parametrize("rows, inner, columns, group", [(40, 1 << 20, 20, 128), (33, (1 << 20) + 2080, 7, 32)])
def test_int4_matmul_of_long_rows(gpu_client, rows, inner, columns, group):
    # rows too long for tiles in the scratch of allocation-free executions; as exact as whole numbers below 2^24 are
    module, ins = vp.int4_case(rows, inner, columns, group, "bf16", zeros=True, out_dtype="f32", exact=True, seed=rows)
    given = [torch.from_numpy(np.array(i.data).view(np.int16 if i.data.dtype == np.uint16 else i.data.dtype)).cuda() for i in ins]
    y = torch.full((rows, columns), 7.0, device="cuda")
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    assert " few" in exe.describe_plan()
    exe.execute_into([(g.data_ptr(), g.nbytes) for g in given], [(y.data_ptr(), y.nbytes)], torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert np.array_equal(y.double().cpu().numpy(), oo.int4_matmul(vp.values(ins), {})[0])


def test_int4_matmul_of_the_longest_rows(gpu_client):
    rows, inner, columns = 17, 1 << 22, 33
    weight = torch.full((columns, inner // 2), 0x88, dtype=torch.uint8, device="cuda")
    weight[::4, -1] = 0x98                                            # the last value 1, the others 0
    weight[1::4] = 0x89                                               # 1, 0, 1, 0, ...
    x = torch.arange(1, rows + 1, device="cuda").bfloat16()[:, None].expand(rows, inner).contiguous()
    x[:, -1] = 5
    scale = torch.full((columns, inner // 32), 0.5, dtype=torch.bfloat16, device="cuda")
    y = torch.full((rows, columns), 7.0, device="cuda")
    exe = gpu_client.compile(pjrt.Program.mlir(operators.int4_matmul_module(rows=rows, inner=inner, columns=columns, group=32, out_dtype="f32")))
    exe.execute_into([(g.data_ptr(), g.nbytes) for g in (x, weight, scale)], [(y.data_ptr(), y.nbytes)],
                     torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = torch.zeros_like(y)
    want[:, ::4] = 2.5
    want[:, 1::4] = torch.arange(1, rows + 1, device="cuda").float()[:, None] * (inner // 4)
    assert torch.equal(y, want)
