"""The operators that verify drafted tokens without a GPU: the oracle against other forms, front-ends, plans and aliasing,
packing, and what is refused."""
import numpy as np
import pytest

from oracle import operators as oo
from ryft_amd import operators, pjrt
from tests import operator_programs as op
from tests import verify_programs as vp
from tests.test_operators import INVALID, UNIMPLEMENTED, refused


# ------------------------------------------------------------------------------------------------ oracle
def test_oracle_of_a_chain_is_causal_attention():
    # a tree without branches is a text: ancestors are the tokens before
    for window in (0, 5):
        module, ins = vp.tree_case([5, 1, 40], [9, 6, 44], 4, 2, 8, 4, "f32", window=window, seed=2)
        x = vp.values(ins)
        chain = [vp.ancestor_words([j - 1 for j in range(n)], 2) for n in (5, 1, 40)]
        x[6] = np.concatenate(chain).astype(np.int64)
        got, = oo.tree_attention(x, op.config_of(module))
        if window:  # the window ends the committed tokens alone: only queries that reach none of the tree's behind it compare
            want, = oo.paged_attention(x[:6], {"scale": 8 ** -0.5, "window": window})
            assert np.allclose(got[:5], want[:5], atol=1e-12) and np.allclose(got[5:10], want[5:10], atol=1e-12)
        else:
            want, = oo.paged_attention(x[:6], {"scale": 8 ** -0.5})
            assert np.allclose(got, want, atol=1e-12)


def test_oracle_of_a_branch_is_the_branch_alone():
    # a leaf's output is that of its path from the root as a text of its own
    r = np.random.RandomState(5)
    parents = vp.random_tree(12, r, wide=True)
    module, ins = vp.tree_case([12], [20], 2, 1, 8, 4, "f32", seed=3)
    x = vp.values(ins)
    x[6] = vp.ancestor_words(parents, 1).astype(np.int64)
    got, = oo.tree_attention(x, op.config_of(module))
    q, kc, vc, table, _, _, _ = x
    flat = [np.stack([c[table[0, p // 4], :, p % 4] for p in range(20)]) for c in (kc, vc)]
    for leaf in range(12):
        path = [leaf]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        keep = list(range(8)) + [8 + j for j in path]
        for h in range(2):
            s = flat[0][keep, 0] @ q[leaf, h] * 8 ** -0.5
            p = np.exp(s - s.max())
            assert np.allclose(got[leaf, h], p @ flat[1][keep, 0] / p.sum(), atol=1e-6)


def test_oracle_acceptance_by_hand():
    # node: 0 root, 1 and 2 its children (equal tokens: the lower), 3 under 1, 4 under 2, 5 under 3
    tokens, parents = np.array([9, 7, 7, 5, 6, 4]), np.array([-1, 0, 0, 1, 2, 3])
    targets, slots, starts = np.array([7, 5, 6, 8, 1, 2]), np.array([10, 11, 2, 3, 4, 5]), np.array([0, 6])
    cache = np.arange(12.0).reshape(3, 1, 4, 1)
    counts, emitted, path, moved = oo.tree_accept([tokens, parents, targets, slots, starts, cache], {})
    assert counts.tolist() == [3] and path.tolist() == [0, 1, 3, -1, -1, -1] and emitted.tolist() == [7, 5, 8, -1, -1, -1]
    want = cache.copy()
    want[0, 0, 2, 0] = 3.0  # node 3's slot 3 to node 2's slot 2
    assert np.array_equal(moved, want)


def test_oracle_int4_against_dequantised_weights():
    r = np.random.RandomState(1)
    w = r.randn(6, 64) * 0.3
    for zeros in (False, True):
        q, scale, zero = operators.quantize_int4(w, 16, zeros)
        back = oo.int4_matmul([np.eye(64), q.astype(np.int64), scale.astype(np.float64), zero.astype(np.int64)], {})[0].T
        # off by half a step; without zero points the magnitudes fit 7 steps, with them the zero's rounding moves the ends by
        # up to half a step more
        assert (np.abs(back - w) <= (1.001 if zeros else 0.501) * np.repeat(scale, 16, axis=1)).all()


def test_pack_and_quantize():
    q = operators.pack_int4(np.array([[1, 2, 15, 0]]))
    assert q.tolist() == [[0x21, 0x0F]] and q.dtype == np.uint8
    for bad in ([[1, 2, 3]], [[16, 0]], [[-1, 0]]):
        with pytest.raises(ValueError):
            operators.pack_int4(np.array(bad))
    q, scale, zero = operators.quantize_int4(np.zeros((2, 8)), 4)
    assert (scale == 0).all() and (zero == 8).all() and (q == 0x88).all()
    with pytest.raises(ValueError):
        operators.quantize_int4(np.zeros((2, 8)), 3)


# ------------------------------------------------------------------------------------------------ front-ends and plans
MODULES = {
    "tree_attention": lambda: vp.tree_case([5, 2], [20, 9], 4, 2, 64, 16, "f16", window=7, softcap=30.0)[0],
    "tree_accept": lambda: vp.accept_case([5, 2], 2, 2, 64, 16, "bf16")[0],
    "int4_matmul": lambda: vp.int4_case(3, 64, 10, 32, "bf16", zeros=True, out_dtype="f32")[0],
}


@pytest.mark.parametrize("name", MODULES)
@pytest.mark.parametrize("order", ["sorted", "declared"])
def test_bytecode_gives_the_same_plan(compile_client, monkeypatch, name, order):
    module = MODULES[name]()
    want = compile_client.compile(pjrt.Program.mlir(module)).describe_plan()
    assert f": {name} " in want
    code = op.to_bytecode(module, monkeypatch, order)
    assert compile_client.compile(pjrt.Program.mlir(code)).describe_plan() == want


def decoder(**kw):
    return operators.decoder_module(tokens=7, sequences=3, vocab=512, layers=2, d_model=256, q_heads=4, kv_heads=2, head_dim=64,
                                    ffn=512, pages=12, page_size=16, pages_per_sequence=4, **kw)


def test_caches_are_moved_in_place(compile_client):
    plan = compile_client.compile(pjrt.Program.mlir(MODULES["tree_accept"]())).describe_plan()
    assert "result 3 <- parameter 5 (in place)" in plan and "result 4 <- parameter 6 (in place)" in plan
    # appended to, read by attention and moved by one program: one buffer for each cache, and no copy but the parameter's own,
    # which an execution that donates it skips
    module, _ = decoder(tree_words=1, int4_group=32)
    plan = compile_client.compile(pjrt.Program.mlir(module)).describe_plan()
    assert plan.count("(in place)") == 4 and plan.count(": copy ") == 4
    assert plan.count(": tree_attention ") == 2 and plan.count(": tree_accept ") == 1 and plan.count(": int4_matmul ") == 8
    assert plan.index(": tree_accept ") > plan.rindex(": tree_attention ") and plan.index(": tree_accept ") > plan.index(": sample ")


def test_int4_matmul_leaves_room_for_other_temporaries(compile_client):
    # allocation-free executions have 64 MiB for all temporaries: beside a large one a product takes less, in more goes
    def plan(rows, columns):
        x, w, s = f"tensor<{rows}x4096xbf16>", f"tensor<{columns}x2048xui8>", f"tensor<{columns}x32xbf16>"
        y, v, t = f"tensor<{rows}x{columns}xf32>", f"tensor<8x{columns // 2}xui8>", f"tensor<8x{columns // 128}xf32>"
        z = f"tensor<{rows}x8xf32>"
        exe = compile_client.compile(pjrt.Program.mlir(
            f"module {{\n  func.func @main(%x: {x}, %w: {w}, %s: {s}, %v: {v}, %t: {t}) -> {z} {{\n"
            + operators.int4_matmul("%y", [("%x", x), ("%w", w), ("%s", s)], y)
            + operators.int4_matmul("%z", [("%y", y), ("%v", v), ("%t", t)], z) + f"    return %z : {z}\n  }}\n}}\n"))
        return exe.describe_plan(), exe.executable().memory_statistics()["temp_size_in_bytes"]

    text, temp = plan(1024, 14336)
    assert " rows=384" in text and 58_720_256 < temp <= 64 << 20
    text, temp = plan(1024, 4096)
    assert " rows=1024" in text and temp <= 64 << 20


def test_a_cache_read_after_the_move_is_copied(compile_client):
    # the attention does not feed the choices: it may come after the move, so the move gets a buffer of its own
    c, q, i, s, w = "tensor<3x2x16x64xbf16>", "tensor<5x4x64xbf16>", "tensor<5xi32>", "tensor<2xi32>", "tensor<5x1xi32>"
    f, k, tab, one = "tensor<32xf32>", "tensor<5x2x64xbf16>", "tensor<1x3xi32>", "tensor<1xi32>"
    append = operators.rope_append("%r", [("%q", q), ("%k", k), ("%v", k), ("%i", i), ("%i", i), ("%f", f), ("%a", c), ("%b", c)])
    tree = operators.tree_attention("%o", [("%r#0", q), ("%r#1", c), ("%r#2", c), ("%tab", tab), ("%s", s), ("%n", one), ("%w", w)], scale=0.1)
    move = operators.tree_accept("%x", [("%i", i)] * 4 + [("%s", s), ("%r#1", c), ("%r#2", c)], 5, 1)
    params = ", ".join(f"%{n}: {t}" for n, t in (("q", q), ("k", k), ("v", k), ("i", i), ("f", f), ("tab", tab), ("s", s), ("n", one), ("w", w)))
    module = (f"module {{\n  func.func @main({params}, %a: {c} {{tf.aliasing_output = 1 : i32}}, %b: {c} {{tf.aliasing_output = 2 : i32}}) -> "
              f"({q}, {c}, {c}) {{\n{append}{move}{tree}    return %o, %x#3, %x#4 : {q}, {c}, {c}\n  }}\n}}\n")
    plan = compile_client.compile(pjrt.Program.mlir(module)).describe_plan()
    lines = plan.split("\n")
    moved = next(n for n, ln in enumerate(lines) if ": tree_accept " in ln)
    assert sum(": copy " in ln for ln in lines[:moved]) == 4  # the parameters into the appended caches, those into the moved ones


# ------------------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("name, old, new, words", [
    ("tree_attention", "tensor<7x1xi32>", "tensor<6x1xi32>", ["visible"]),
    ("tree_attention", "tensor<7x1xi32>", "tensor<7x0xi32>", ["words"]),
    ("tree_attention", "tensor<7x1xi32>", "tensor<7x1xf32>", ["visible"]),
    ("tree_attention", "softcap = 3.e+01 : f32", "causal = true", ["unknown", "causal"]),
    ("tree_attention", "window = 7 : i64", "window = -1 : i64", ["window"]),
    ("tree_attention", "tensor<7x4x64xf16>", "tensor<7x5x64xf16>", ["5 query heads"]),
    ("tree_accept", "tensor<3xi32>", "tensor<4xi32>", ["result 0"]),
    ("tree_accept", "tensor<3x2x16x64xbf16>", "tensor<3x2x16x64xi32>", ["i32"]),
    ("tree_accept", "tensor<3x2x16x64xbf16>", "tensor<3x2x16x512xbf16>", ["head dim"]),
    ("int4_matmul", "10x32xui8", "10x31xui8", ["weight"]),
    ("int4_matmul", "3x64xbf16", "3x63xbf16", ["even number"]),
    ("int4_matmul", "3x64xbf16", "3x64xi32", ["i32"]),
    ("int4_matmul", "10x2xbf16", "10x3xbf16", ["groups"]),
    ("int4_matmul", "10x2xbf16", "10x64xbf16", ["groups"]),
    ("int4_matmul", "10x2xbf16", "10x2xf16", ["scale"]),
    ("int4_matmul", "10x2xui8", "10x2xi32", ["zero"]),
    ("int4_matmul", "-> tensor<3x10xf32>", "-> tensor<3x10xf16>", ["result"]),
    ("int4_matmul", "backend_config = {}", "backend_config = {group = 32 : i64}", ["unknown"]),
])
def test_refusals_of_types_and_config(compile_client, name, old, new, words):
    module = MODULES[name]()
    assert old in module, module
    refused(compile_client, module.replace(old, new), UNIMPLEMENTED if words == ["i32"] else INVALID, *words)


def test_refusals_of_the_caches(compile_client):
    m = MODULES["tree_accept"]()
    c = "tensor<3x2x16x64xbf16>"
    # caches of two types, and a result too few
    other = m.replace(f"%arg6: {c}", "%arg6: tensor<3x2x16x64xf16>").replace(f"{c}, {c}) ->", f"{c}, tensor<3x2x16x64xf16>) ->")
    refused(compile_client, other, INVALID)
    many = vp.accept_case([2], 257, 1, 4, 4, "f32")[0]
    refused(compile_client, many, INVALID, "257 caches")
    plan = compile_client.compile(pjrt.Program.mlir(vp.accept_case([2], 256, 1, 4, 4, "f32")[0])).describe_plan()
    assert "caches=256" in plan and plan.count("(in place)") == 256
    refused(compile_client, MODULES["tree_attention"]().replace(", %arg6)", ")").replace(", tensor<7x1xi32>) ->", ") ->"), INVALID, "7 operands")
