"""The decoding operators without a GPU at the edges of their definitions."""
import numpy as np
import pytest

from ryft_amd import operators, pjrt
from tests import operator_programs as op


def attention(client, **kw):
    args = dict(tokens=3, sequences=2, q_heads=4, kv_heads=2, head_dim=64, pages=5, page_size=16, pages_per_sequence=4, scale=0.125)
    args.update(kw)
    return client.compile(pjrt.Program.mlir(operators.paged_attention_module(**args)))


# ------------------------------------------------------------------------------------------------ config
def test_every_finite_f32_is_a_scale_and_a_cap(compile_client):
    # the largest, as its shortest decimal form (which is larger than it is)
    most = float(np.finfo(np.float32).max)
    for kw in (dict(softcap=most), dict(scale=most), dict(scale=-most), dict(softcap=1e-45), dict(scale=1e-45)):
        attention(compile_client, **kw)
    for kw in (dict(softcap=np.inf), dict(scale=np.inf), dict(scale=-np.inf), dict(scale=np.nan)):
        with pytest.raises(pjrt.PjrtError) as e:
            attention(compile_client, **kw)
        assert e.value.code == pjrt.ErrorCode.INVALID_ARGUMENT and "out of range" in str(e.value)


def test_other_targets_are_not_implemented_whatever_their_config(compile_client, monkeypatch):
    # as a program from another front-end has them: an opaque string, a value that no operator here takes
    module = operators.sample_module(rows=3, vocab=100)
    other = module.replace("@ryft.sample", "@Sharding")
    opaque = [other.replace("api_version = 4 : i32, backend_config = {}", f"api_version = 2 : i32, backend_config = {c}")
              for c in ('"opaque"', '{shape = [1, 2]}', '{k = "v"}')]
    for text in [other] + opaque:
        assert "Sharding" in text
        with pytest.raises(pjrt.PjrtError) as e:
            compile_client.compile(pjrt.Program.mlir(text))
        assert e.value.code == pjrt.ErrorCode.UNIMPLEMENTED and "'Sharding'" in str(e.value)
    code = op.to_bytecode(other.replace("backend_config = {}", "backend_config = {k = 3 : i64}"), monkeypatch)
    with pytest.raises(pjrt.PjrtError) as e:
        compile_client.compile(pjrt.Program.mlir(code))
    assert e.value.code == pjrt.ErrorCode.UNIMPLEMENTED and "'Sharding'" in str(e.value)


# ------------------------------------------------------------------------------------------------ chains of appends
def plan(client, *args, **kw):
    return client.compile(pjrt.Program.mlir(op.append_chain(*args, **kw)[0])).describe_plan()


@pytest.mark.parametrize("steps", [1, 2, 3])
@pytest.mark.parametrize("first", ["queries", "caches"])
def test_a_chain_of_appends_is_one_buffer(compile_client, steps, first):
    # one copy a cache, which an execution that donates it skips, whichever result the plan begins with
    last = [f"%r{steps - 1}#1", f"%r{steps - 1}#2"]
    queries = [f"%r{n}#0" for n in range(steps)]
    text = plan(compile_client, steps, returns=queries + last if first == "queries" else last[::-1] + queries)
    assert text.count(": rope_append ") == steps and text.count(": copy") == 2
    assert text.count("(in place)") == 2 and "(own buffer)" not in text


def test_what_else_reads_a_cache_keeps_it(compile_client):
    # the cache between two appends as a result of its own, or one value as both caches: buffers of their own, copied
    c = "tensor<2x2x16x64xbf16>"
    text = plan(compile_client, 2, returns=["%r0#1", "%r1#1", "%r1#2"])
    assert "result 1 <- parameter 1 (own buffer)" in text and "result 2 <- parameter 2 (in place)" in text
    module, _ = op.append_chain(1, returns=["%r0#1", "%r0#2"])
    both = module.replace("%kc, %vc)", "%e, %e)").replace("    %r0:3", f"    %e = stablehlo.add %kc, %vc : {c}\n    %r0:3")
    assert both.count("%e") == 3
    text = compile_client.compile(pjrt.Program.mlir(both)).describe_plan()
    assert text.count(": copy") == 2 and "(in place)" not in text


# ------------------------------------------------------------------------------------------------ workspaces
@pytest.mark.parametrize("d, sequences, heads, keys", [(128, 1, (8, 1), 32768), (64, 1, (4, 2), 32768), (128, 2, (16, 2), 100016), (128, 4, (32, 8), 16384),
                                                       (64, 9, (16, 4), 2048)], ids=str)
def test_ranges_of_keys_take_room_for_the_parts_there_can_be(compile_client, d, sequences, heads, keys):
    # a part is 128 rows of d values, a maximum and a sum; a tile is cut into 128 ranges at most, each of 128 keys at least,
    # and a launch has two workgroups a CU, three for heads of 64
    exe = attention(compile_client, tokens=sequences * 5, sequences=sequences, q_heads=heads[0], kv_heads=heads[1], head_dim=d,
                    pages=8, pages_per_sequence=keys // 16)
    tiles = (sequences * 5 * (heads[0] // heads[1]) // 128 + sequences) * heads[1]
    parts = min(512 if d == 128 else 768, tiles * min(128, keys // 128))
    temp = exe.executable().memory_statistics()["temp_size_in_bytes"]
    assert 0 <= temp - parts * 128 * (d + 2) * 4 <= 16384, temp


def test_room_for_long_contexts_leaves_decoding_steps_to_their_kernel(compile_client):
    # (told by the workspace: two parts of 16 rows a workgroup; ranges of keys, 128 rows, only for the fewest sequences)
    few = lambda d: 2 * 512 * 16 * (d + 2) * 4  # noqa: E731
    for d, sequences, heads, keys, want in ((128, 4, (32, 8), 32768, True), (64, 2, (16, 8), 65536, True), (128, 1, (32, 8), 16368, True),
                                            (128, 1, (32, 8), 16384, False), (64, 4, (8, 2), 131072, False)):
        exe = attention(compile_client, tokens=sequences, sequences=sequences, q_heads=heads[0], kv_heads=heads[1], head_dim=d,
                        pages=8, pages_per_sequence=keys // 16)
        temp = exe.executable().memory_statistics()["temp_size_in_bytes"]
        assert (temp == few(d)) == want, (d, sequences, heads, keys, temp)
