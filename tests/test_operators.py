"""The decoding operators without a GPU: the oracle against closed forms, the front-ends (text, generic text, bytecode),
plans and aliasing, and what is refused."""
import math

import numpy as np
import pytest
import torch

from oracle import operators as oo
from oracle import stablehlo as sh
from ryft_amd import operators, pjrt
from tests import operator_programs as op


# ------------------------------------------------------------------------------------------------ oracle
def test_oracle_rotation_is_a_complex_product():
    for interleaved in (False, True):
        module, ins = op.append_case(5, 3, 2, 16, 12, 4, 3, "f32", norm=False, interleaved=interleaved, start=1000)
        x = op.values(ins)
        q, kc, vc = oo.rope_append(x, op.config_of(module))
        rot, half = 12, 6
        for got, src in ((q, x[0]), (np.stack([kc[s // 4, :, s % 4] for s in x[4]]), x[1])):
            a, b = (src[..., 0:rot:2], src[..., 1:rot:2]) if interleaved else (src[..., :half], src[..., half:rot])
            z = (a + 1j * b) * np.exp(1j * x[3][:, None, None] * x[5])
            ga, gb = (got[..., 0:rot:2], got[..., 1:rot:2]) if interleaved else (got[..., :half], got[..., half:rot])
            assert np.allclose(ga, z.real, atol=1e-12) and np.allclose(gb, z.imag, atol=1e-12)
            assert np.array_equal(got[..., rot:], src[..., rot:])
        for t, s in enumerate(x[4]):
            assert np.array_equal(vc[s // 4, :, s % 4], x[2][t])


def test_oracle_attention_matches_torch():
    module, ins = op.attention_case([3, 1, 4], [9, 6, 4], 4, 2, 8, 4, "f32")
    x = op.values(ins)
    got, = oo.paged_attention(x, op.config_of(module))
    q, kc, vc, table, starts, lengths = x
    for b in range(3):
        n, length = int(starts[b + 1] - starts[b]), int(lengths[b])
        rows = [(int(table[b, p // 4]), p % 4) for p in range(length)]
        k, v = (np.stack([c[pg, :, o] for pg, o in rows], axis=1) for c in (kc, vc))
        want = torch.nn.functional.scaled_dot_product_attention(
            torch.tensor(q[starts[b]:starts[b + 1]].transpose(1, 0, 2)),
            torch.tensor(np.repeat(k, 2, axis=0)), torch.tensor(np.repeat(v, 2, axis=0)),
            attn_mask=torch.tensor(np.arange(length)[None] <= (length - n + np.arange(n))[:, None]), scale=8 ** -0.5)
        assert np.allclose(got[starts[b]:starts[b + 1]], want.numpy().transpose(1, 0, 2), atol=1e-6)


def test_oracle_sample_borders():
    # weights 4, 2, 1, 1 (of 8) at temperature 1, in the order of the indices 1, 3, 0, 2
    x = np.log([[1.0, 4.0, 1.0, 2.0]])

    def token(u, k=0, p=1.0, m=0.0, t=1.0):
        (tok,), (lp,) = oo.sample([x, np.array([t]), np.array([k]), np.array([p]), np.array([m]), np.array([u])], {})
        return int(tok), lp

    assert [token(u)[0] for u in (0.0, 0.124, 0.126, 0.624, 0.626, 0.749, 0.751, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [token(u, k=2)[0] for u in (0.0, 0.66, 0.67, 0.999)] == [1, 1, 3, 3]
    assert [token(u, k=3)[0] for u in (0.0, 0.2, 0.9)] == [0, 1, 3]         # of two equal ones the lower index
    assert [token(u, p=0.5)[0] for u in (0.0, 0.999)] == [1, 1]              # 4/8 reach one half
    assert [token(u, p=0.51)[0] for u in (0.0, 0.7)] == [1, 3]
    assert [token(u, p=0.76)[0] for u in (0.0, 0.2, 0.999)] == [0, 1, 3]
    assert [token(u, m=0.5)[0] for u in (0.0, 0.7)] == [1, 3]
    assert token(0.9, t=0.0) == (1, 0.0) and token(0.9, p=0.0) == (1, 0.0)
    assert math.isclose(token(0.7, k=2)[1], math.log(1 / 3))


# ------------------------------------------------------------------------------------------------ front-ends and plans
MODULES = {
    "rope_append": lambda: op.append_case(5, 4, 2, 64, 64, 16, 3, "bf16", norm=True, interleaved=False)[0],
    "paged_attention": lambda: op.attention_case([2, 1], [20, 5], 4, 2, 64, 16, "f16", window=7, softcap=30.0, slopes=True)[0],
    "sample": lambda: operators.sample_module(rows=3, vocab=100, dtype="bf16"),
}


@pytest.mark.parametrize("name", MODULES)
@pytest.mark.parametrize("order", ["sorted", "declared"])
def test_bytecode_gives_the_same_plan(compile_client, monkeypatch, name, order):
    module = MODULES[name]()
    want = compile_client.compile(pjrt.Program.mlir(module)).describe_plan()
    assert f": {name} " in want
    code = op.to_bytecode(module, monkeypatch, order)
    assert compile_client.compile(pjrt.Program.mlir(code)).describe_plan() == want


def test_generic_text_gives_the_same_plan(compile_client):
    module = MODULES["paged_attention"]()
    line = next(ln for ln in module.split("\n") if "custom_call" in ln)
    head, rest = line.split("custom_call @")
    target, rest = rest.split("(", 1)
    args, rest = rest.split(") {", 1)
    attrs, types = rest.rsplit("} : ", 1)
    generic = (f'    %0 = "stablehlo.custom_call"({args}) <{{call_target_name = "{target}", has_side_effect = false, '
               f'{attrs}, operand_layouts = []}}> : {types}')
    assert (compile_client.compile(pjrt.Program.mlir(module.replace(line, generic))).describe_plan()
            == compile_client.compile(pjrt.Program.mlir(module)).describe_plan())


def test_caches_are_updated_in_place(compile_client):
    plan = compile_client.compile(pjrt.Program.mlir(MODULES["rope_append"]())).describe_plan()
    assert "result 1 <- parameter 6 (in place)" in plan and "result 2 <- parameter 7 (in place)" in plan
    # the attention over the updated caches leaves them in place; a reader of the old cache does not
    module, _ = operators.decoder_module(tokens=7, sequences=3, vocab=512, layers=2, d_model=256, q_heads=4, kv_heads=2,
                                         head_dim=64, ffn=512, pages=12, page_size=16, pages_per_sequence=4)
    plan = compile_client.compile(pjrt.Program.mlir(module)).describe_plan()
    assert plan.count("(in place)") == 4 and plan.count(": rope_append ") == 2 and plan.count(": paged_attention ") == 2
    c, q = "tensor<3x2x16x64xbf16>", "tensor<5x4x64xbf16>"
    old = MODULES["rope_append"]().replace(f"-> ({q}, {c}, {c}) {{", f"-> ({q}, {c}, {c}, {c}) {{")
    old = old.replace(f"    return %0#0, %0#1, %0#2 : {q}, {c}, {c}",
                      f"    %n = stablehlo.negate %arg6 : {c}\n    return %0#0, %0#1, %0#2, %n : {q}, {c}, {c}, {c}")
    plan = compile_client.compile(pjrt.Program.mlir(old)).describe_plan()
    # (the old keys are read by the negation before anything writes the new ones, or from a buffer of their own)
    assert "result 2 <- parameter 7 (in place)" in plan
    lines = plan.split("\n")
    where = {n: next(i for i, ln in enumerate(lines) if n in ln) for n in (": elementwise", ": rope_append")}
    assert where[": elementwise"] < where[": rope_append"] or "result 1 <- parameter 6 (own buffer)" in plan


def test_projection_slices_are_read_in_place(compile_client):
    module, _ = operators.decoder_module(tokens=7, sequences=3, vocab=512, layers=1, d_model=256, q_heads=4, kv_heads=2,
                                         head_dim=64, ffn=512, pages=12, page_size=16, pages_per_sequence=4)
    plan = compile_client.compile(pjrt.Program.mlir(module)).describe_plan()
    assert "transpose_copy" not in plan and "slice" not in plan


# ------------------------------------------------------------------------------------------------ refusals
def refused(client, module, code, *words):
    with pytest.raises(pjrt.PjrtError) as e:
        client.compile(pjrt.Program.mlir(module))
    assert e.value.code == code, e.value
    for w in words:
        assert w in str(e.value), (w, str(e.value))


INVALID, UNIMPLEMENTED = pjrt.ErrorCode.INVALID_ARGUMENT, pjrt.ErrorCode.UNIMPLEMENTED


def test_refusals_of_the_call(compile_client):
    m = MODULES["sample"]()
    refused(compile_client, m.replace("@ryft.sample", "@somebody.else"), UNIMPLEMENTED, "somebody.else")
    refused(compile_client, m.replace("backend_config = {}", "backend_config = {k = 3 : i64}"), INVALID, "unknown", "'k'")
    refused(compile_client, m.replace("backend_config = {}", 'backend_config = "k=3"'), INVALID, "dictionary")
    refused(compile_client, m.replace("backend_config = {}", "backend_config = {k = [1]}"), INVALID)
    refused(compile_client, m.replace("api_version = 4 : i32", "has_side_effect = true"), UNIMPLEMENTED, "side effects")
    refused(compile_client, m.replace(", %arg5)", ")").replace(", tensor<3xf32>) ->", ") ->"), INVALID)


@pytest.mark.parametrize("name, old, new, words", [
    ("sample", "3x100xbf16", "3x100xi32", ["i32"]),
    ("sample", "-> (tensor<3xi32>, tensor<3xf32>)", "-> (tensor<3xi32>, tensor<4xf32>)", ["result 1"]),
    ("rope_append", "tensor<32xf32>", "tensor<33xf32>", ["inv_freq"]),
    ("rope_append", "tensor<3x2x16x64xbf16>", "tensor<3x4x16x64xbf16>", ["key cache"]),
    ("rope_append", "tensor<3x2x16x64xbf16>", "tensor<3x2x16x64xf16>", ["key cache"]),
    ("rope_append", "tensor<64xbf16>", "tensor<64xf32>", ["q_weight"]),
    ("rope_append", "eps = 1.e-05 : f32", "eps = -1.0 : f32", ["eps"]),
    ("paged_attention", "tensor<2xi32>", "tensor<4xi32>", ["page_table"]),
    ("paged_attention", "tensor<4xf32>", "tensor<5xf32>", ["slopes"]),
    ("paged_attention", "window = 7 : i64", "window = -1 : i64", ["window"]),
    ("paged_attention", "window = 7 : i64", "window = 7.5 : f32", ["window"]),
    ("paged_attention", "softcap = 3.e+01 : f32", "softcap = 0x7FC00000 : f32", ["softcap"]),
    ("paged_attention", "3x4x64xf16", "3x5x64xf16", ["5 query heads"]),
])
def test_refusals_of_types_and_config(compile_client, name, old, new, words):
    module = MODULES[name]()
    assert old in module, module
    code = UNIMPLEMENTED if words == ["i32"] else INVALID
    refused(compile_client, module.replace(old, new), code, *words)


def test_head_dim_and_norm_refusals(compile_client):
    refused(compile_client, op.append_case(1, 1, 1, 512, 64, 16, 1, "bf16", norm=False, interleaved=False)[0], INVALID, "head dim")
    refused(compile_client, op.attention_case([1], [3], 1, 1, 264, 16, "f32")[0], INVALID, "head dim")
    m = op.append_case(1, 1, 1, 64, 64, 16, 1, "bf16", norm=False, interleaved=False)[0]
    refused(compile_client, m.replace("magnitude", "eps = 1e-6 : f32, magnitude"), INVALID, "eps")


def test_execute_into_needs_a_device(compile_client):
    exe = compile_client.compile(pjrt.Program.mlir(MODULES["sample"]()))
    with pytest.raises(pjrt.PjrtError) as e:
        exe.execute_into([(256, 4)] * 6, [(256, 4)] * 2)
    assert e.value.code == pjrt.ErrorCode.FAILED_PRECONDITION
