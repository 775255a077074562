"""Plans of programs with int4_matmul and the workspace that they take, without a GPU: allocation-free executions have 64 MiB
for all temporaries of a program."""
import numpy as np
import pytest

from ryft_amd import operators, pjrt
from tests.test_operators import INVALID, refused

SCRATCH = 64 << 20


def planned(client, module):
    exe = client.compile(pjrt.Program.mlir(module))
    return exe.describe_plan(), exe.executable().memory_statistics()["temp_size_in_bytes"]


def products(text):
    """Each int4_matmul's line, without its number."""
    return [ln.split(": ", 1)[1] for ln in text.split("\n") if ": int4_matmul " in ln]


# ------------------------------------------------------------------------------------------------ one product
@pytest.mark.parametrize("rows, inner, group", [(17, 1 << 22, 32), (17, 1 << 22, 128), (300, 1 << 20, 128), (2048, 1 << 21, 64)])
def test_rows_too_long_for_tiles_go_without_a_workspace(compile_client, rows, inner, group):
    text, temp = planned(compile_client, operators.int4_matmul_module(rows=rows, inner=inner, columns=64, group=group))
    assert " few" in text and temp == 0


@pytest.mark.parametrize("rows, inner, columns, group", [(17, 1 << 18, 64, 128), (512, 25600, 4096, 32), (1024, 52352, 4096, 128),
                                                         (40, 1 << 19, 300, 32), (100_000, 64, 4096, 32)])
def test_one_product_fits_the_scratch(compile_client, rows, inner, columns, group):
    text, temp = planned(compile_client, operators.int4_matmul_module(rows=rows, inner=inner, columns=columns, group=group))
    assert " tile=" in text and 0 < temp <= SCRATCH


# ------------------------------------------------------------------------------------------------ groups that do not fit
@pytest.mark.parametrize("inner, group", [(128, 48), (100, 33), (64, 128), (64, 3), (96, 0), (96, -32), (96, 1)])
def test_modules_refuse_groups_that_rows_are_not_cut_into(inner, group):
    # (128 values in groups of 48 would become a program with two groups of 64)
    with pytest.raises(ValueError, match="groups"):
        operators.int4_matmul_module(rows=2, inner=inner, columns=10, group=group)


@pytest.mark.parametrize("what, size", [("int4_group", 96), ("int4_group", 31), ("int4_group", -32), ("ffn", 200), ("tree_words", -1)])
def test_decoders_refuse_groups_that_rows_are_not_cut_into(what, size):
    cfg = dict(tokens=4, sequences=2, vocab=64, layers=1, d_model=128, q_heads=2, kv_heads=1, head_dim=64, ffn=192, pages=2, page_size=16,
               pages_per_sequence=1, int4_group=32)
    operators.decoder_module(**cfg)
    with pytest.raises(ValueError, match="groups|words"):
        operators.decoder_module(**{**cfg, what: size})


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 1e40])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_refuses_what_is_not_finite(zeros, bad):
    w = np.ones((2, 8))
    w[1, 3] = bad
    with pytest.raises(ValueError, match="finite"):
        operators.quantize_int4(w, 4, zeros)


def test_quantize_refuses_what_is_no_matrix():
    for w in (np.ones(8), np.ones((2, 2, 8))):
        with pytest.raises(ValueError):
            operators.quantize_int4(w, 4)


# ------------------------------------------------------------------------------------------------ trees that are too large
def test_tree_accept_refuses_trees_that_steps_of_a_workgroup_would_leave(compile_client):
    # nodes are counted in 32 bits, 256 at a time: a tree of 2^31 - 1 would be counted past that
    most = 1 << 30
    text, _ = planned(compile_client, operators.tree_accept_module(tokens=most, sequences=1))
    assert f"tokens={most}" in text
    for tokens in (most + 1, (1 << 31) - 1):
        refused(compile_client, operators.tree_accept_module(tokens=tokens, sequences=1), INVALID, "too many tokens")


# ------------------------------------------------------------------------------------------------ beside other temporaries
def beside(rows, inner, columns, group, other, dtype="bf16", product=True):
    """A product and a temporary of `other` f32 rows of 4096 beside it: a matrix product that another one reads. Or that alone."""
    x, w, s = f"tensor<{rows}x{inner}x{dtype}>", f"tensor<{columns}x{inner // 2}xui8>", f"tensor<{columns}x{inner // group}x{dtype}>"
    y, a, b = f"tensor<{rows}x{columns}xf32>", f"tensor<{other}x64xf32>", "tensor<64x4096xf32>"
    t, c, z = f"tensor<{other}x4096xf32>", "tensor<4096x64xf32>", f"tensor<{other}x64xf32>"
    dot = "stablehlo.dot_general {}, {}, contracting_dims = [1] x [0] : ({}, {}) -> {}"
    return (f"module {{\n  func.func @main(%x: {x}, %w: {w}, %s: {s}, %a: {a}, %b: {b}, %c: {c}) -> ({y}, {z}) {{\n"
            + (operators.int4_matmul("%y", [("%x", x), ("%w", w), ("%s", s)], y) if product else f"    %y = stablehlo.constant dense<0.0> : {y}\n")
            + f"    %t = {dot.format('%a', '%b', a, b, t)}\n    %z = {dot.format('%t', '%c', t, c, z)}\n"
            + f"    return %y, %z : {y}, {z}\n  }}\n}}\n")


def alone(client, rows, inner, columns, group, dtype="bf16"):
    text, temp = planned(client, operators.int4_matmul_module(rows=rows, inner=inner, columns=columns, group=group, dtype=dtype, out_dtype="f32"))
    return products(text)[0], temp


def test_a_product_takes_what_others_leave(compile_client):
    size = (256, 14336, 4096, 64, "f16")
    line, temp = alone(compile_client, *size)
    assert " parts=8" in line and temp < SCRATCH
    for other in (1, 1024, 1536, 1792, 2560, 3584, 3840, 4064):
        text, together = planned(compile_client, beside(*size[:4], other, size[4]))
        rest = planned(compile_client, beside(*size[:4], other, size[4], product=False))[1]
        if temp + rest <= SCRATCH:
            assert products(text) == [line]                           # nothing to save
            continue
        assert together <= SCRATCH, (other, text)
        left, mine = SCRATCH - rest, together - rest
        if left > 24 << 20:                                           # the rows take 8 MiB, each of four ranges of K 4
            assert " rows=256" in products(text)[0] and mine >= 23 << 20, (other, text)
        elif left > 4 << 20:
            assert " tile=" in products(text)[0], text
    assert other == 4064 and " few" in products(text)[0]              # (half a MiB is left)


def test_a_product_keeps_its_plan_where_none_would_fit(compile_client):
    size = (256, 14336, 4096, 64, "f16")
    line, _ = alone(compile_client, *size)
    text, temp = planned(compile_client, beside(*size[:4], 4200, size[4]))
    assert temp > SCRATCH and products(text) == [line]


def test_a_decoder_keeps_its_plans_where_none_would_fit(compile_client):
    cfg = dict(tokens=256, d_model=4096, ffn=14336)
    module, _ = operators.decoder_module(sequences=16, vocab=1024, layers=1, q_heads=32, kv_heads=8, head_dim=128, pages=64, page_size=16,
                                         pages_per_sequence=4, int4_group=128, tree_words=2, **cfg)
    text, temp = planned(compile_client, module)
    assert temp > SCRATCH
    sizes = [(4096, 6144), (4096, 4096), (4096, 28672), (14336, 4096)]
    assert products(text) == [alone(compile_client, 256, k, n, 128)[0] for k, n in sizes]


def test_products_and_edge_gemms_make_room_together(compile_client):
    # 16 bf16 products of 2432 x 128 x 11520 take 76 MiB of partial sums in the ranges that are estimated fastest; the 4-bit product's
    # parts and rows 60 MB: only with less of both is there room
    x, w, s = "tensor<1024x14336xbf16>", "tensor<4096x7168xui8>", "tensor<4096x112xbf16>"
    y, a, b, z = "tensor<1024x4096xf32>", "tensor<16x2432x11520xbf16>", "tensor<16x11520x128xbf16>", "tensor<16x2432x128xf32>"
    module = (f"module {{\n  func.func @main(%x: {x}, %w: {w}, %s: {s}, %a: {a}, %b: {b}) -> ({y}, {z}) {{\n"
              + operators.int4_matmul("%y", [("%x", x), ("%w", w), ("%s", s)], y)
              + f"    %z = stablehlo.dot_general %a, %b, batching_dims = [0] x [0], contracting_dims = [2] x [1] : ({a}, {b}) -> {z}\n"
              + f"    return %y, %z : {y}, {z}\n  }}\n}}\n")
    text, temp = planned(compile_client, module)
    assert 0 < temp <= SCRATCH and " tile=" in products(text)[0], text
