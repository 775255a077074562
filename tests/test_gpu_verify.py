"""The operators that verify drafted tokens on the GPU against the oracle in 64 bits, through
PJRT_LoadedExecutable_Execute and, where noted, through execute_into.

Tolerances. A result is rounded once to its type: half a step of it, `HALF_STEP`, relative to the value. tree_attention's
are paged_attention's (tests/test_gpu_operators.py), whose kernels it runs with another mask. int4_matmul's sums are f32:
`int4_error` counts their roundings; where a sum is whole numbers below 2^24 it is exact. tree_accept has no roundings."""
import numpy as np
import pytest
import torch  # (before the plugin: both then use one HIP runtime)

from oracle import operators as oo
from oracle import stablehlo as sh
from ryft_amd import operators, pjrt
from tests import operator_programs as op
from tests import verify_programs as vp
from tests.test_gpu_operators import attention_error, close, device_buffers, run, span

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ tree_attention
TREES = {
    # nodes and total lengths of each sequence, query / key heads, head dim, page size, options
    "one": dict(nodes=[1], lengths=[1], heads=(1, 1, 64), page=16),
    "pair": dict(nodes=[2, 2], lengths=[2, 300], heads=(8, 2, 128), page=16),
    "small": dict(nodes=[8, 5, 1, 3], lengths=[100, 5, 700, 64], heads=(8, 8, 128), page=16),
    "small_64": dict(nodes=[8, 5, 1, 16], lengths=[300, 77, 513, 16], heads=(4, 4, 64), page=32),
    "across_blocks": dict(nodes=[16, 15, 9], lengths=[40, 71, 136], heads=(2, 2, 128), page=16),
    "long_few": dict(nodes=[4], lengths=[9001], heads=(4, 1, 128), page=16),
    "wide": dict(nodes=[64, 40, 64], lengths=[700, 41, 64], heads=(8, 2, 128), page=16),
    "wide_64": dict(nodes=[130, 33, 64], lengths=[1030, 33, 200], heads=(6, 3, 64), page=64),
    "odd_group": dict(nodes=[50, 31], lengths=[333, 100], heads=(5, 1, 128), page=16),
    "ranges": dict(nodes=[48], lengths=[6000], heads=(8, 2, 64), page=16),
    "many": dict(nodes=[3] * 70, lengths=[30 + 9 * i for i in range(70)], heads=(4, 2, 64), page=16),
    "window": dict(nodes=[12, 60, 4], lengths=[900, 400, 64], heads=(4, 2, 128), page=16, window=100),
    "window_few": dict(nodes=[3, 4, 2], lengths=[900, 400, 64], heads=(4, 2, 64), page=16, window=70),
    "window_one": dict(nodes=[3, 40], lengths=[200, 100], heads=(2, 2, 64), page=16, window=1),
    "softcap": dict(nodes=[4, 90], lengths=[300, 200], heads=(4, 2, 128), page=16, softcap=5.0, spread=2.0),
    "softcap_few": dict(nodes=[4, 5], lengths=[300, 200], heads=(4, 2, 64), page=16, softcap=5.0, spread=2.0, window=130),
    "random": dict(nodes=[40, 33], lengths=[300, 90], heads=(4, 2, 128), page=16, masks="random"),
    "random_few": dict(nodes=[4, 7], lengths=[300, 20], heads=(2, 2, 64), page=16, masks="random"),
    "random_window": dict(nodes=[30, 3], lengths=[300, 90], heads=(4, 2, 64), page=16, masks="random", window=20),
    "nothing_of_the_tree": dict(nodes=[30, 3], lengths=[300, 3], heads=(4, 2, 64), page=16, masks="none", window=50),
    "all_of_the_tree": dict(nodes=[30, 3], lengths=[300, 90], heads=(4, 2, 128), page=16, masks="all"),
    "past_the_words": dict(nodes=[70, 40], lengths=[300, 90], heads=(4, 2, 64), page=16, words=1),
    "spare_words": dict(nodes=[5, 20], lengths=[300, 90], heads=(4, 2, 128), page=16, words=7),
    "empty": dict(nodes=[0, 1, 0, 3], lengths=[50, 0, 0, 2], heads=(4, 2, 64), page=16, spare=3),
    "before_the_start": dict(nodes=[40, 5], lengths=[10, 0], heads=(4, 2, 128), page=16),
    "before_the_start_few": dict(nodes=[4, 5], lengths=[2, 0], heads=(2, 2, 64), page=16, window=3),
    "odd_pages": dict(nodes=[7, 60], lengths=[300, 131], heads=(4, 2, 128), page=24),
    "page_of_one": dict(nodes=[3, 20], lengths=[70, 20], heads=(2, 1, 64), page=1),
    "bad_pages": dict(nodes=[3, 1, 70, 2], lengths=[300, 10, 200, 64], heads=(4, 2, 128), page=16, bad_pages=True),
    "poison": dict(nodes=[3, 70, 1, 3], lengths=[301, 200, 64, 70], heads=(4, 2, 128), page=16, poison=True),
    "head_80": dict(nodes=[5, 30], lengths=[200, 90], heads=(4, 2, 80), page=16, window=40),
    "head_256": dict(nodes=[5, 30], lengths=[200, 90], heads=(4, 2, 256), page=16, softcap=20.0),
}


def tree(name, dtype):
    c = dict(TREES[name])
    nodes, lengths, (hq, hkv, d), page = (c.pop(k) for k in ("nodes", "lengths", "heads", "page"))
    return vp.tree_case(nodes, lengths, hq, hkv, d, page, dtype, seed=len(name), **c)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("name", TREES)
def test_tree_attention(gpu_client, name, dtype):
    module, ins = tree(name, dtype)
    (got,), _ = run(gpu_client, module, ins, [dtype])
    x = vp.values(ins)
    want, = oo.tree_attention(x, op.config_of(module))
    assert np.isfinite(want).all()
    close(got, want, dtype, attention_error(x, dtype), name)
    nothing = ~want.any(axis=(1, 2))
    assert not got[nothing].any()                                     # rows that see nothing are exactly zero


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(4, 2, 128), (2, 2, 64)], ids=str)
@pytest.mark.parametrize("nodes", [[5, 3], [70, 40]], ids=str)
def test_tree_attention_branches_do_not_see_each_other(gpu_client, nodes, heads, dtype):
    # NaN and infinite keys and values of nodes: only queries below them may show it
    hq, hkv, d = heads
    module, ins = vp.tree_case(nodes, [nodes[0] + 60, nodes[1] + 7], hq, hkv, d, 16, dtype, seed=7)
    x = vp.values(ins)
    kc, vc, table, words = x[1], x[2], x[3], x[6]
    for b, node, junk in ((0, nodes[0] - 2, (np.nan, np.inf)), (1, nodes[1] - 1, (np.inf, np.nan))):
        p = (60, 7)[b] + node
        kc[table[b, p // 16], :, p % 16], vc[table[b, p // 16], :, p % 16] = junk
    ins[1], ins[2] = op.host(kc, dtype), op.host(vc, dtype)
    (got,), _ = run(gpu_client, module, ins, [dtype])
    want, = oo.tree_attention(x, op.config_of(module))
    hit = np.array([int(words[t, j // 32]) >> j % 32 & 1 for t, j in
                    [(t, nodes[0] - 2) for t in range(nodes[0])] + [(nodes[0] + t, nodes[1] - 1) for t in range(nodes[1])]], dtype=bool)
    assert hit.any() and not hit.all()
    close(got[~hit], want[~hit], dtype, attention_error(x, dtype), "others")
    assert np.isfinite(got[~hit]).all() and not np.isfinite(got[hit]).any(axis=2).all()


def test_tree_attention_of_a_chain_is_causal(gpu_client):
    for nodes, lengths in (([6, 3], [200, 70]), ([90, 40], [300, 100])):
        module, ins = vp.tree_case(nodes, lengths, 4, 2, 128, 16, "bf16", seed=1)
        ins[6] = op.host(np.concatenate([vp.ancestor_words([j - 1 for j in range(n)], 3 if nodes[0] > 64 else 1) for n in nodes]), "i32")
        (got,), _ = run(gpu_client, module, ins, ["bf16"])
        text = operators.paged_attention_module(tokens=sum(nodes), sequences=2, q_heads=4, kv_heads=2, head_dim=128, pages=ins[1].dims[0],
                                                page_size=16, pages_per_sequence=ins[3].dims[1], scale=128 ** -0.5)
        (want,), _ = run(gpu_client, text, ins[:6], ["bf16"])
        close(got, want, "bf16", attention_error(vp.values(ins), "bf16"), "chain")


@pytest.mark.parametrize("starts, lengths", [([-5, 30, 20, 60], [3000, 2000, 40]), ([60, 0, 60, 0], [900, 900, 900]),
                                             ([0, 70, 70, 70], [2 ** 31 - 1, -1, 5]), ([10, 20, 5, 2 ** 31 - 1], [100, 0, 2000])], ids=str)
@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 2, 128)], ids=str)
def test_tree_attention_bad_starts_stay_in_bounds(gpu_client, starts, lengths, heads):
    nodes = [20, 20, 20] if heads[0] == 4 else [5, 4, 6]
    module, ins = vp.tree_case(nodes, [3000, 2000, 40], *heads, 16, "bf16", seed=4, masks="random", window=700)
    ins[4], ins[5] = op.host(starts, "i32"), op.host(lengths, "i32")
    (got,), _ = run(gpu_client, module, ins, ["bf16"])
    assert np.isfinite(got).all() and np.abs(got).max() <= np.abs(vp.values(ins)[2]).max()


@pytest.mark.parametrize("nodes", [[4, 2], [50, 40]], ids=str)
def test_tree_attention_past_32_bits(gpu_client, nodes):
    # pages of caches of 4.6 GB each, their last among them, against the same pages in small caches
    pages, hkv, page, d, lengths = 140_000, 8, 16, 128, [300, 90]
    _, ins = vp.tree_case(nodes, lengths, 16, hkv, d, page, "bf16", seed=4)
    small = [torch.from_numpy(np.array(i.data).view(np.int16 if i.data.dtype == np.uint16 else i.data.dtype)).cuda() for i in ins]
    few = small[1].shape[0]
    to = torch.linspace(0, pages - 1, few, device="cuda").round().long()
    big = list(small)
    for n in (1, 2):
        big[n] = torch.zeros((pages, hkv, page, d), dtype=small[n].dtype, device="cuda")
        big[n][to] = small[n]
    big[3] = torch.where((small[3] >= 0) & (small[3] < few), to[small[3].clamp(0, few - 1).long()].int(), small[3])
    got = []
    for x, count in ((small, few), (big, pages)):
        module = operators.tree_attention_module(
            tokens=sum(nodes), sequences=2, q_heads=16, kv_heads=hkv, head_dim=d, pages=count, page_size=page,
            pages_per_sequence=x[3].shape[1], words=x[6].shape[1], dtype="bf16", scale=d ** -0.5)
        exe = gpu_client.compile(pjrt.Program.mlir(module))
        out = torch.zeros_like(x[0])
        exe.execute_into([(t.data_ptr(), t.nbytes) for t in x], [(out.data_ptr(), out.nbytes)], torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        got.append(out)
    assert int((got[0] != 0).sum()) > 0 and torch.equal(got[0], got[1])


# ------------------------------------------------------------------------------------------------ int4_matmul
SIZES = [
    # rows, inner, columns, group
    (1, 64, 1, 32), (1, 256, 16, 128), (1, 4096, 100, 128), (2, 96, 17, 32), (3, 320, 33, 64), (5, 2, 3, 2), (7, 100, 9, 50),
    (16, 512, 48, 128), (17, 1024, 64, 64), (33, 160, 31, 32), (16, 384, 70, 96), (8, 384, 65, 192), (64, 512, 257, 256),
    (65, 1152, 130, 128), (100, 608, 200, 32), (129, 256, 300, 64), (300, 640, 129, 128), (257, 128, 1000, 128), (12, 3232, 40, 32),
    (31, 8192, 24, 128), (200, 4128, 72, 32), (513, 96, 64, 48),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("zeros", [False, True], ids=["eight", "zeros"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_int4_matmul(gpu_client, size, zeros, dtype):
    seed = sum(size) + zeros
    # (scales in f32 and results in f32 with 16-bit rows, each in some of the cases)
    scale_dtype, out_dtype = (dtype, "f32")[seed % 2], (dtype, "f32")[seed // 2 % 2]
    module, ins = vp.int4_case(*size, dtype, zeros=zeros, scale_dtype=scale_dtype, out_dtype=out_dtype, seed=seed)
    (got,), _ = run(gpu_client, module, ins, [out_dtype])
    x = vp.values(ins)
    want, = oo.int4_matmul(x, {})
    close(got, want, out_dtype, vp.int4_error(x) + 2.0 ** -25, "y")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_int4_matmul_of_whole_numbers_is_exact(gpu_client, size, dtype):
    # every value has a place that shows: sums are whole numbers (of quarters) below 2^24
    module, ins = vp.int4_case(*size, dtype, zeros=True, out_dtype="f32", exact=True, seed=sum(size))
    (got,), _ = run(gpu_client, module, ins, ["f32"])
    want, = oo.int4_matmul(vp.values(ins), {})
    assert np.array_equal(got, want)


def test_int4_matmul_zero_points_past_15(gpu_client):
    # a zero point is a byte: any of its values
    module, ins = vp.int4_case(5, 256, 40, 64, "bf16", zeros=True, out_dtype="f32", exact=True, seed=3)
    ins[3] = vp.host(np.resize(np.arange(0, 256, 5), ins[3].dims), "ui8")
    (got,), _ = run(gpu_client, module, ins, ["f32"])
    assert np.array_equal(got, oo.int4_matmul(vp.values(ins), {})[0])


@pytest.mark.parametrize("rows, inner", [(3, 512), (40, 512), (300, 512), (4, 96)])
def test_int4_matmul_keeps_infinities_in_their_rows(gpu_client, rows, inner):
    module, ins = vp.int4_case(rows, inner, 70, 32, "bf16", seed=5)
    x = vp.values(ins)
    x[0][1, 5], x[0][rows - 1, inner - 1] = np.nan, np.inf
    ins[0] = op.host(x[0], "bf16")
    (got,), _ = run(gpu_client, module, ins, ["bf16"])
    want, = oo.int4_matmul(vp.values(ins), {})
    clean = [r for r in range(rows) if r not in (1, rows - 1)]
    assert not np.isfinite(got[[1, rows - 1]]).any()
    close(got[clean], want[clean], "bf16", vp.int4_error([x[0][clean], *x[1:]]), "others")


# more tiles of the weight than workgroups, steps of x in registers or not, and rows that are prepared in two goes
MORE_SIZES = [
    (1, 1024, 8201, 64), (2, 4096, 8230, 128), (3, 2048, 4300, 32), (4, 1152, 4500, 96), (5, 2304, 4200, 768), (9, 8192, 4111, 64),
    (16, 4000, 4128, 32), (16, 4096, 8300, 128), (7, 5152, 4333, 32), (13, 8224, 4111, 32), (8, 160, 12321, 32), (300, 32768, 70, 128),
    (270, 30752, 33, 32), (40, 20480, 300, 64),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True], ids=["eight", "zeros"])
@pytest.mark.parametrize("size", MORE_SIZES, ids=str)
def test_int4_matmul_of_more_tiles(gpu_client, size, zeros, dtype):
    module, ins = vp.int4_case(*size, dtype, zeros=zeros, out_dtype="f32", exact=True, seed=sum(size) + zeros)
    (got,), _ = run(gpu_client, module, ins, ["f32"])
    assert np.array_equal(got, oo.int4_matmul(vp.values(ins), {})[0])


@pytest.mark.parametrize("dtype, factor", [("bf16", 2.0 ** 100), ("bf16", 2.0 ** -100), ("f16", 2.0 ** 14), ("f16", 2.0 ** -24)])
@pytest.mark.parametrize("size", [(1, 4096, 300, 128), (16, 2304, 4200, 64), (3, 2048, 4300, 32), (40, 512, 300, 64), (300, 640, 129, 128)], ids=str)
def test_int4_matmul_of_large_and_small_values(gpu_client, size, dtype, factor):
    # whole numbers times a power of two: as exact as they are, f16's subnormal numbers among them
    module, ins = vp.int4_case(*size, dtype, zeros=True, out_dtype="f32", exact=True, seed=sum(size))
    ins[0] = op.host(vp.values(ins)[0] * factor, dtype)
    (got,), _ = run(gpu_client, module, ins, ["f32"])
    assert np.array_equal(got, oo.int4_matmul(vp.values(ins), {})[0])


def test_int4_matmul_of_slices(gpu_client):
    # rows of the weight, scales and zero points that begin anywhere within larger tensors, and a slice of x
    r = np.random.RandomState(4)
    x, w = r.randint(-3, 4, (9, 200)), r.randint(0, 256, (41, 80))
    scale, zero = 2.0 ** r.randint(-2, 3, (41, 5)), r.randint(0, 16, (41, 5))
    module = """
module @slices {
  func.func public @main(%x: tensor<9x200xf16>, %w: tensor<41x80xui8>, %s: tensor<41x5xf16>, %z: tensor<41x5xui8>) -> tensor<5x33xf32> {
    %0 = stablehlo.slice %x [3:8, 7:167] : (tensor<9x200xf16>) -> tensor<5x160xf16>
    %1 = stablehlo.slice %w [5:38, 0:80] : (tensor<41x80xui8>) -> tensor<33x80xui8>
    %2 = stablehlo.slice %s [5:38, 0:5] : (tensor<41x5xf16>) -> tensor<33x5xf16>
    %3 = stablehlo.slice %z [5:38, 0:5] : (tensor<41x5xui8>) -> tensor<33x5xui8>
    %4 = stablehlo.custom_call @ryft.int4_matmul(%0, %1, %2, %3) {api_version = 4 : i32, backend_config = {}} : (tensor<5x160xf16>, tensor<33x80xui8>, tensor<33x5xf16>, tensor<33x5xui8>) -> tensor<5x33xf32>
    return %4 : tensor<5x33xf32>
  }
}
"""
    ins = [op.host(x, "f16"), vp.host(w, "ui8"), op.host(scale, "f16"), vp.host(zero, "ui8")]
    (got,), _ = run(gpu_client, module, ins, ["f32"])
    want, = oo.int4_matmul([x[3:8, 7:167].astype(float), w[5:38], scale[5:38], zero[5:38]], {})
    assert np.array_equal(got, want)


@pytest.mark.parametrize("rows", [1, 5, 20])
def test_int4_matmul_past_32_bits(gpu_client, rows):
    # a weight of 8.6 GB that is 0 but for its last rows and some between
    inner, columns, group = 16384, (1 << 20) + 3, 128
    weight = torch.full((columns, inner // 2), 0x88, dtype=torch.uint8, device="cuda")
    scale = torch.ones((columns, inner // group), dtype=torch.bfloat16, device="cuda")
    some = [0, 1 << 19, 700_001, columns - 2, columns - 1]
    for k, n in enumerate(some):
        weight[n] = 0x99 + 0x11 * k
    x = torch.arange(rows, device="cuda").bfloat16()[:, None].expand(rows, inner).contiguous() + 1
    y = torch.full((rows, columns), 7.0, dtype=torch.float32, device="cuda")
    exe = gpu_client.compile(pjrt.Program.mlir(operators.int4_matmul_module(rows=rows, inner=inner, columns=columns, group=group,
                                                                            out_dtype="f32")))
    exe.execute_into([(t.data_ptr(), t.nbytes) for t in (x, weight, scale)], [(y.data_ptr(), y.nbytes)],
                     torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = torch.zeros_like(y)
    for k, n in enumerate(some):
        want[:, n] = x[:, 0].float() * (k + 1) * inner
    assert torch.equal(y, want)


def test_int4_matmul_of_no_rows(gpu_client):
    module, ins = vp.int4_case(0, 64, 10, 32, "bf16")
    (got,), _ = run(gpu_client, module, ins, ["bf16"])
    assert got.shape == (0, 10)


# ------------------------------------------------------------------------------------------------ tree_accept
ACCEPT = {
    "one": dict(nodes=[1], caches=1, heads=(1, 64), page=16, dtype="bf16"),
    "small": dict(nodes=[8, 1, 5, 12], caches=2, heads=(2, 64), page=16, dtype="bf16"),
    "deep": dict(nodes=[60, 33, 64], caches=4, heads=(8, 128), page=16, dtype="f16", vocab=2),
    "chain_of_one_token": dict(nodes=[300, 40], caches=2, heads=(1, 64), page=16, dtype="bf16", vocab=1),
    "wide": dict(nodes=[64, 256], caches=3, heads=(2, 128), page=32, dtype="f32", wide=True),
    "no_caches": dict(nodes=[20, 9], caches=0, heads=(1, 1), page=4, dtype="bf16"),
    "empty": dict(nodes=[0, 3, 0, 0, 2], caches=1, heads=(2, 64), page=16, dtype="bf16", spare=5),
    "no_sequences": dict(nodes=[], caches=1, heads=(2, 64), page=16, dtype="bf16", spare=300),
    "many": dict(nodes=[7] * 300, caches=2, heads=(1, 64), page=16, dtype="bf16", vocab=2),
    "odd_heads": dict(nodes=[30, 20], caches=2, heads=(3, 7), page=5, dtype="bf16", vocab=2),
    "odd_heads_32": dict(nodes=[30, 20], caches=1, heads=(3, 3), page=1, dtype="f32", vocab=2),
    "heads_of_12": dict(nodes=[30, 20], caches=1, heads=(2, 12), page=4, dtype="f16", vocab=2),
    "bad_parents": dict(nodes=[40, 30, 60], caches=2, heads=(2, 64), page=16, dtype="bf16", bad_parents=True, vocab=2),
    "bad_slots": dict(nodes=[40, 30, 60], caches=2, heads=(2, 64), page=16, dtype="bf16", bad_slots=True, vocab=1),
    "past_the_words_of_a_workgroup": dict(nodes=[9000, 5], caches=1, heads=(1, 8), page=64, dtype="bf16", vocab=2),
}


@pytest.mark.parametrize("name", ACCEPT)
def test_tree_accept(gpu_client, name):
    c = dict(ACCEPT[name])
    nodes, caches, heads, page, dtype = (c.pop(k) for k in ("nodes", "caches", "heads", "page", "dtype"))
    module, ins = vp.accept_case(nodes, caches, *heads, page, dtype, seed=len(name), **c)
    got, _ = run(gpu_client, module, ins, ["i32"] * 3 + [dtype] * caches)
    want = oo.tree_accept(vp.values(ins), {})
    for what, g, w in zip(["counts", "emitted", "path"] + ["cache"] * caches, got, want):
        assert np.array_equal(g, w), what


def test_tree_accept_of_many_caches(gpu_client):
    # as many results as a call may have
    module, ins = vp.accept_case([20, 9], 256, 1, 8, 16, "f16", vocab=1, wide=True, seed=6)
    got, _ = run(gpu_client, module, ins, ["i32"] * 3 + ["f16"] * 256)
    want = oo.tree_accept(vp.values(ins), {})
    for n, (g, w) in enumerate(zip(got, want)):
        assert np.array_equal(g, w), n


def test_tree_accept_of_one_cache_twice(gpu_client):
    # each result gets its own copy; donated, the parameter's memory becomes the first one's
    module, ins = vp.accept_case([30, 20], 2, 2, 64, 16, "bf16", vocab=1, wide=True, seed=2)
    module = module.replace("%arg6)", "%arg5)")
    x = vp.values(ins)
    want = oo.tree_accept(x[:6] + [x[5]], {})
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    for donated in (False, True):
        bufs = device_buffers(gpu_client, ins)
        out = exe.execute([[pjrt.ExecutionInput(b, donatable=donated and n == 5) for n, b in enumerate(bufs)]])[0]
        out.done.await_()
        for n, (g, w) in enumerate(zip(out.outputs, want)):
            got = sh.from_raw(g.to_numpy(), "i32" if n < 3 else "bf16")
            assert np.array_equal(got, w), (donated, n)
        assert bufs[5].is_deleted() == donated


def test_tree_accept_past_32_bits(gpu_client):
    # a cache of 4.6 GB, moved in place: rows at its end, the path 0, 2, 3 of a tree whose every choice is token 1
    pages, hkv, page, d = 140_000, 8, 16, 128
    cache = torch.zeros((pages, hkv, page, d), dtype=torch.bfloat16, device="cuda")
    slots = [pages * page - 1 - 37 * i for i in range(4)]
    for i, slot in enumerate(slots):
        cache[slot // page, :, slot % page] = i + 1
    module = operators.tree_accept_module(tokens=4, sequences=1, caches=1, pages=pages, kv_heads=hkv, page_size=page, head_dim=d)
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    words = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ins = [words(0, 2, 1, 1), words(-1, 0, 0, 2), words(1, 1, 1, 7), words(*slots), words(0, 4), cache]
    outs = [words(9), words(9, 9, 9, 9), words(9, 9, 9, 9)]
    exe.execute_into([(t.data_ptr(), t.nbytes) for t in ins], [(t.data_ptr(), t.nbytes) for t in outs + [cache]],
                     torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert [o.tolist() for o in outs] == [[3], [1, 1, 7, -1], [0, 2, 3, -1]]
    for slot, want in zip(slots, (1, 3, 4, 4)):
        assert (cache[slot // page, :, slot % page] == want).all(), slot
    assert int((cache[:70_000] != 0).sum()) == 0


def test_tree_accept_bad_starts_stay_in_bounds(gpu_client):
    module, ins = vp.accept_case([20, 20, 20], 2, 2, 64, 16, "bf16", vocab=2, seed=2)
    for starts in ([-5, 30, 20, 60], [60, 0, 60, 0], [10, 20, 5, 2 ** 31 - 1], [-2 ** 31, -1, -1, -1]):
        ins[4] = op.host(starts, "i32")
        got, _ = run(gpu_client, module, ins, ["i32"] * 3 + ["bf16"] * 2)
        assert (got[0] >= 0).all() and (got[0] <= 60).all()


# ------------------------------------------------------------------------------------------------ as a program runs them
PROGRAMS = {
    "tree_few": lambda: tree("small_64", "bf16"),
    "tree_wide": lambda: tree("wide", "bf16"),
    "tree_ranges": lambda: tree("ranges", "f16"),
    "int4_one": lambda: vp.int4_case(1, 2048, 512, 128, "bf16", seed=1),
    "int4_some": lambda: vp.int4_case(40, 2048, 512, 64, "f16", zeros=True, seed=2),
    "int4_many": lambda: vp.int4_case(500, 2048, 512, 128, "bf16", seed=3),
    "int4_any": lambda: vp.int4_case(4, 96, 50, 48, "f32", seed=4),
}


@pytest.mark.parametrize("name", PROGRAMS)
def test_replayed_from_a_graph(gpu_client, name):
    # captured on a stream of torch's, replayed with eager executions of the same executable in between
    module, ins = PROGRAMS[name]()
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    bufs = device_buffers(gpu_client, ins)
    ref = exe.execute([bufs])[0]
    ref.done.await_()
    want = ref.outputs[0].to_numpy()
    out = gpu_client.uninitialized_buffer(ref.outputs[0].element_type(), ref.outputs[0].dimensions())
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        exe.execute_into([span(b) for b in bufs], [span(out)], torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.to_numpy(), want), i
        again = exe.execute([bufs])[0]
        again.done.await_()
        assert np.array_equal(again.outputs[0].to_numpy(), want), i


@pytest.mark.parametrize("names", [("int4_some", "int4_many"), ("tree_few", "int4_some"), ("tree_ranges", "int4_many")], ids=str)
def test_two_graphs_in_turn(gpu_client, names):
    # they share the scratch memory; each replay leaves nothing of it for the next
    made = []
    for name in names:
        module, ins = PROGRAMS[name]()
        exe = gpu_client.compile(pjrt.Program.mlir(module))
        bufs = device_buffers(gpu_client, ins)
        ref = exe.execute([bufs])[0]
        ref.done.await_()
        out = gpu_client.uninitialized_buffer(ref.outputs[0].element_type(), ref.outputs[0].dimensions())
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            exe.execute_into([span(b) for b in bufs], [span(out)], torch.cuda.current_stream().cuda_stream)
        made.append((graph, out, ref.outputs[0].to_numpy(), exe, bufs))
    for i in range(4):
        for graph, *_ in made:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, want, *_ in made:
            assert np.array_equal(out.to_numpy(), want), i


def test_tree_accept_replayed_in_place(gpu_client):
    # the caches are parameter and result at once, and change with every replay; a copy of them is moved eagerly beside
    module, ins = vp.accept_case([30, 20, 40], 2, 2, 64, 16, "bf16", vocab=1, wide=True, seed=3)
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    bufs, mine = device_buffers(gpu_client, ins), device_buffers(gpu_client, ins)
    outs = [gpu_client.uninitialized_buffer(pjrt.BufferType.S32, d) for d in ((3,), (90,), (90,))]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        exe.execute_into([span(b) for b in bufs], [span(o) for o in outs + bufs[5:]], torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        ref = exe.execute([[pjrt.ExecutionInput(b, donatable=n >= 5) for n, b in enumerate(mine)]])[0]
        ref.done.await_()
        assert all(mine[n].is_deleted() for n in (5, 6))
        mine[5:] = ref.outputs[3:]
        for got, want in zip(outs + bufs[5:], ref.outputs):
            assert np.array_equal(got.to_numpy(), want.to_numpy())


@pytest.mark.parametrize("name", PROGRAMS)
def test_results_repeat(gpu_client, name):
    # no result depends on the order in which workgroups come
    module, ins = PROGRAMS[name]()
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    bufs = device_buffers(gpu_client, ins)
    first = None
    for _ in range(6):
        out = exe.execute([bufs])[0]
        out.done.await_()
        got = out.outputs[0].to_numpy()
        assert first is None or np.array_equal(got, first)
        first = got


# ------------------------------------------------------------------------------------------------ together
def test_a_step_that_verifies_drafts(gpu_client):
    """Prompts of two sequences through a two-layer decoder with 4-bit weights, then steps that verify trees of drafted tokens.
    A node's choice does not depend on the nodes beside and below it, so drafts that are the choices of an earlier run of the
    same step are accepted; path, counts and moved caches are the oracle's, and the next step goes on from them."""
    cfg = dict(vocab=300, layers=2, d_model=128, q_heads=4, kv_heads=2, head_dim=64, ffn=192, pages=12, page_size=16,
               pages_per_sequence=6, int4_group=32)
    r = np.random.RandomState(11)
    texts = [list(r.randint(0, 300, n)) for n in (21, 7)]
    table = r.permutation(12).reshape(2, 6)
    weights = {}

    def step(module, params, small, caches, donate=True):
        ins = []
        for name, shape, dt in params:
            if name in small:
                ins.append(vp.host(np.asarray(small[name]).reshape(shape), dt))
                continue
            if name not in weights:
                if dt == "ui8":
                    w = r.randn(shape[0], 2 * shape[1]) * (2 * shape[1]) ** -0.5
                    q, scale, _ = operators.quantize_int4(w, 32)
                    weights[name], weights[f"{name}_scale"] = vp.host(q, "ui8"), op.host(scale, "bf16")
                else:
                    x = 1 + 0.1 * r.randn(*shape) if len(shape) == 1 else r.randn(*shape)
                    weights[name] = op.host(np.zeros(shape) if name.endswith(("_k", "_v")) else x, dt)
            ins.append(weights[name])
        names = [p[0] for p in params]
        where = [i for i, n in enumerate(names) if n.startswith("l") and n.endswith(("_k", "_v"))]
        exe = gpu_client.compile(pjrt.Program.mlir(module))
        bufs, vals = device_buffers(gpu_client, ins), vp.values(ins)
        for i, c in zip(where, caches or []):
            bufs[i], vals[i] = c, sh.from_raw(c.to_numpy(), "bf16")
        out = exe.execute([[pjrt.ExecutionInput(b, donatable=donate and i in where) for i, b in enumerate(bufs)]])[0]
        out.done.await_()
        return out.outputs, vals

    def inputs(ids, positions, places, rows):
        seq = np.concatenate([np.full(len(n), b) for b, n in enumerate(ids)])
        at = np.concatenate(places)
        return {"ids": np.concatenate(ids), "positions": np.concatenate(positions), "slots": table[seq, at // 16] * 16 + at % 16,
                "table": table, "starts": np.cumsum([0] + [len(n) for n in ids]), "lengths": [p[-1] + 1 for p in places],
                "temperature": np.zeros(rows), "top_k": np.zeros(rows), "top_p": np.ones(rows), "min_p": np.zeros(rows),
                "uniform": np.zeros(rows), "inv_freq": 10000.0 ** (-np.arange(32) / 32)}

    module, params = operators.decoder_module(tokens=28, sequences=2, **cfg)
    every = [np.arange(len(t)) for t in texts]
    out, vals = step(module, params, {**inputs(texts, every, every, 2), "last": [20, 27]}, None)
    for c, (w, _) in zip(out[2:], sh.evaluate(module, vals)[2:]):
        assert sh.rel_error(sh.from_raw(c.to_numpy(), "bf16"), w) < 3e-2
    caches = out[2:]
    for t, c in zip(texts, out[0].to_numpy()):
        t.append(int(c))

    up, depth = [-1, 0, 0, 2, 2, 4], np.array([0, 1, 1, 2, 2, 3])
    module, params = operators.decoder_module(tokens=12, sequences=2, tree_words=1, **cfg)
    plan = gpu_client.compile(pjrt.Program.mlir(module)).describe_plan()
    assert ": int4_matmul " in plan and ": tree_attention " in plan and ": tree_accept " in plan
    for _ in range(3):
        drafts = [[t[-1]] + [(t[-1] + j) % 300 for j in range(1, 6)] for t in texts]
        base = [len(t) - 1 for t in texts]                             # the root is the last token, not in the caches yet
        fixed = {"parents": up * 2, "visible": np.concatenate([vp.ancestor_words(up, 1)] * 2)}
        shape = ([b + depth for b in base], [b + np.arange(6) for b in base], 12)
        chosen = []
        for child in (2, 4):                                           # the draft becomes what its parent's choice was
            out, _ = step(module, params, {**inputs(drafts, *shape), **fixed}, caches, donate=False)
            chosen.append(out[0].to_numpy())
            for b, d in enumerate(drafts):
                d[child] = int(chosen[-1][6 * b + up[child]])
                for j in range(child):                                 # (and no lower sibling has the same)
                    if up[j] == up[child] and d[j] == d[child]:
                        d[j] = (d[j] + 1) % 300
        small = {**inputs(drafts, *shape), **fixed}
        out, vals = step(module, params, small, caches)
        targets, _, counts, emitted, path = (o.to_numpy() for o in out[:5])
        for b in range(2):
            assert targets[6 * b] == chosen[0][6 * b] and targets[6 * b + 2] == chosen[1][6 * b + 2]
            assert path[6 * b:6 * b + 3].tolist() == [0, 2, 4] and counts[b] >= 3
        names = ["ids", "parents", "slots", "starts"]
        want = oo.tree_accept([np.asarray(small[n]) for n in names[:2]] + [targets] + [np.asarray(small[n]) for n in names[2:]], {})
        for got, w in zip((counts, emitted, path), want):
            assert np.array_equal(got, w)
        # the caches: what the oracle appends, moved along the path that was taken
        alone = [np.full(12, -1) if n == "parents" else v for (n, _, _), v in zip(params, vals)]  # (no node is reached)
        appended = sh.evaluate(module, alone)[5:]
        moved = oo.tree_accept([np.asarray(small["ids"]), np.asarray(small["parents"]), targets, np.asarray(small["slots"]),
                                np.asarray(small["starts"])] + [w for w, _ in appended], {})[3:]
        for c, w in zip(out[5:], moved):
            assert sh.rel_error(sh.from_raw(c.to_numpy(), "bf16"), w) < 3e-2
        caches = out[5:]
        for b, t in enumerate(texts):
            t += [int(v) for v in emitted[6 * b:6 * b + counts[b]]]
