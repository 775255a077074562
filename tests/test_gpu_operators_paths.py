"""The decoding operators at the sizes where their kernels change: batches of more than a wavefront of sequences, tiles cut
into ranges of keys, rows that many workgroups share, vocabularies beyond the chunks. Tolerances as in
test_gpu_operators.py."""
import numpy as np
import pytest
import torch  # (before the plugin: both then use one HIP runtime)

from oracle import operators as oo
from ryft_amd import operators, pjrt
from tests import operator_programs as op
from tests.test_gpu_operators import attention_error, check_sample, close, device_buffers, run, span, sync

pytestmark = pytest.mark.gpu


def spread(n, most, seed):
    return [int(v) for v in np.random.RandomState(seed).randint(1, most + 1, n)]


# ------------------------------------------------------------------------------------------------ paged_attention
ATTENTION = {
    # a decoding step, sequences found 64 at a time, some without keys
    "step_150": dict(new=[1] * 150, lengths=[0, 1] + spread(148, 250, 1), heads=(4, 2, 64), page=16),
    "step_150_128": dict(new=[1] * 150, lengths=spread(150, 150, 2), heads=(8, 2, 128), page=16, window=100, slopes=True),
    "step_uneven": dict(new=[0, 1, 2, 0, 9] * 14, lengths=[7, 300, 3, 0, 130] * 14, heads=(4, 4, 64), page=32, spare=5),
    # few long sequences: one tile in as many ranges as there can be, and in fewer
    "long_one": dict(new=[1], lengths=[20001], heads=(4, 1, 128), page=32),
    "long_ragged": dict(new=[1, 1, 2], lengths=[17000, 40, 3000], heads=(4, 2, 64), page=16, softcap=30.0),
    "long_just_short": dict(new=[1], lengths=[16100], heads=(2, 1, 64), page=16),
    # chunks over long contexts
    "ranges": dict(new=[5], lengths=[6001], heads=(8, 1, 128), page=16),
    "ranges_ragged": dict(new=[17, 2, 20, 1], lengths=[5000, 300, 64, 2000], heads=(5, 1, 64), page=16),
    "ranges_window": dict(new=[33, 40], lengths=[3000, 2500], heads=(4, 2, 128), page=16, window=700, slopes=True),
    "ranges_not_causal": dict(new=[20, 3], lengths=[2000, 900], heads=(8, 2, 64), page=64, causal=False, softcap=30.0),
    "ranges_bad_pages": dict(new=[20, 9], lengths=[2000, 1100], heads=(4, 1, 128), page=16, bad_pages=True),
    "ranges_poison": dict(new=[20, 9], lengths=[2001, 1100], heads=(4, 1, 64), page=16, poison=True),
    "ranges_two_tiles": dict(new=[70], lengths=[4000], heads=(4, 1, 64), page=16),
    "ranges_70": dict(new=spread(70, 9, 3), lengths=[9 + n for n in spread(70, 800, 4)], heads=(8, 1, 64), page=16),
    "ranges_70_uneven": dict(new=[0, 12, 3, 1, 0] * 14, lengths=[7, 900, 3, 0, 0] * 14, heads=(8, 1, 128), page=16, spare=3),
    # prompts whose tiles alone fill the chip
    "prompts": dict(new=spread(34, 50, 5), lengths=[50 + n for n in spread(34, 200, 6)], heads=(16, 16, 64), page=16),
    "prompts_window": dict(new=spread(34, 50, 7), lengths=[50 + n for n in spread(34, 300, 8)], heads=(16, 16, 64), page=16,
                           window=100),
    "prompts_not_causal": dict(new=[0, 33, 1, 50] * 10, lengths=[5, 40, 0, 90] * 10, heads=(16, 16, 64), page=16, causal=False),
    "prompts_no_keys": dict(new=[17, 40] * 20, lengths=[0, 3] * 20, heads=(16, 16, 64), page=16, spare=2),
    "prompts_100": dict(new=spread(66, 50, 9), lengths=[50 + n for n in spread(66, 60, 10)], heads=(8, 8, 64), page=16),
    # pages of one key: the table's entries are read 64 at a time
    "page_of_one_step": dict(new=[1, 1], lengths=[700, 65], heads=(2, 2, 64), page=1),
    "page_of_one_chunk": dict(new=[40, 3], lengths=[600, 129], heads=(2, 1, 128), page=1),
    "page_of_three": dict(new=[40, 1], lengths=[600, 131], heads=(2, 2, 64), page=3),
    # nothing at all
    "nothing": dict(new=[0, 0, 0], lengths=[0, 5, 0], heads=(4, 2, 64), page=16, spare=4),
    "nothing_seen": dict(new=[1, 1], lengths=[0, 0], heads=(4, 2, 128), page=16),
    # scores within half the cap, and far beyond it
    "cap_far": dict(new=[70, 1], lengths=[200, 90], heads=(4, 2, 64), page=16, softcap=50.0),
    "cap_near": dict(new=[70, 1], lengths=[200, 90], heads=(4, 2, 64), page=16, softcap=0.5, spread=2.0),
}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("name", ATTENTION)
def test_paged_attention(gpu_client, name, dtype):
    c = dict(ATTENTION[name])
    new, lengths, (hq, hkv, d), page = (c.pop(k) for k in ("new", "lengths", "heads", "page"))
    module, ins = op.attention_case(new, lengths, hq, hkv, d, page, dtype, seed=len(name), **c)
    (got,), _ = run(gpu_client, module, ins, [dtype])
    x = op.values(ins)
    want, = oo.paged_attention(x, op.config_of(module))
    assert np.isfinite(want).all()
    close(got, want, dtype, attention_error(x, dtype), name)
    assert not got[sum(new):].any()
    unseen = ~want.any(axis=(1, 2))
    assert not got[unseen].any()


@pytest.mark.parametrize("softcap", [0.0, 4.0])
@pytest.mark.parametrize("scale", [-0.125, 0.0])
def test_paged_attention_scales(gpu_client, scale, softcap):
    for new, lengths in (([1, 2], [300, 70]), ([60, 9], [300, 70])):
        _, ins = op.attention_case(new, lengths, 4, 2, 64, 16, "bf16", seed=12)
        module = operators.paged_attention_module(
            tokens=sum(new), sequences=2, q_heads=4, kv_heads=2, head_dim=64, pages=ins[1].dims[0], page_size=16,
            pages_per_sequence=ins[3].dims[1], scale=scale, softcap=softcap)
        (got,), _ = run(gpu_client, module, ins, ["bf16"])
        x = op.values(ins)
        want, = oo.paged_attention(x, op.config_of(module))
        close(got, want, "bf16", attention_error(x, "bf16"), (scale, softcap))


@pytest.mark.parametrize("new, lengths", [([1, 1, 1], [300, 20, 70]), ([1], [20000]), ([30, 5], [900, 40])], ids=str)
def test_paged_attention_strided_queries(gpu_client, new, lengths):
    # queries as a slice of one projection, read in place
    hq, hkv, d, t = 4, 2, 64, sum(new)
    whole, ins = op.attention_case(new, lengths, hq, hkv, d, 16, "bf16", seed=13)
    r = np.random.RandomState(14)
    a = op.host(r.randn(t, hq + 2 * hkv, d), "bf16")
    ty = {k: f"tensor<{'x'.join(map(str, v.dims))}x{e}>" for k, v, e in
          (("a", a, "bf16"), ("c", ins[1], "bf16"), ("t", ins[3], "i32"), ("s", ins[4], "i32"), ("l", ins[5], "i32"))}
    q = f"tensor<{t}x{hq}x{d}xbf16>"
    call = operators.paged_attention("%o", [("%q", q), ("%k", ty["c"]), ("%v", ty["c"]), ("%t", ty["t"]), ("%s", ty["s"]), ("%l", ty["l"])],
                                     scale=d ** -0.5)
    module = (f"module {{\n  func.func @main(%a: {ty['a']}, %k: {ty['c']}, %v: {ty['c']}, %t: {ty['t']}, %s: {ty['s']}, %l: {ty['l']}) -> {q} {{\n"
              f"    %q = stablehlo.slice %a [0:{t}, {hkv}:{hkv + hq}, 0:{d}] : ({ty['a']}) -> {q}\n{call}    return %o : {q}\n  }}\n}}\n")
    (got,), _ = run(gpu_client, module, [a] + ins[1:], ["bf16"])
    x = op.values([a] + ins[1:])
    want, = oo.paged_attention([x[0][:, hkv:hkv + hq], *x[1:]], op.config_of(module))
    close(got, want, "bf16", attention_error(x, "bf16"), "strided")


@pytest.mark.parametrize("starts, lengths", [([-5, 30, 20, 60], [3000, 2000, 40]), ([60, 0, 60, 0], [900, 900, 900]),
                                             ([0, 70, 70, 70], [2 ** 31 - 1, -1, 5]), ([10, 20, 5, 2 ** 31 - 1], [100, 0, 2000])], ids=str)
def test_paged_attention_bad_starts_of_prompts_stay_in_bounds(gpu_client, starts, lengths):
    # starts that decrease or leave the queries: some rows belong to several sequences or to none, and every row is written
    module, ins = op.attention_case([20, 20, 20], [3000, 2000, 40], 4, 2, 64, 16, "bf16", seed=4)
    ins[4], ins[5] = op.host(starts, "i32"), op.host(lengths, "i32")
    (got,), _ = run(gpu_client, module, ins, ["bf16"])
    assert np.isfinite(got).all() and np.abs(got).max() <= np.abs(op.values(ins)[2]).max()


@pytest.mark.parametrize("new, lengths, heads", [([1] * 70, [70 + 5 * i for i in range(70)], (4, 2, 64)), ([1], [20000], (8, 1, 128)),
                                                 ([40, 40], [3000, 700], (8, 2, 128))], ids=["step", "long", "chunk"])
def test_paged_attention_replayed_from_a_graph(gpu_client, new, lengths, heads):
    module, ins = op.attention_case(new, lengths, *heads, 16, "bf16", seed=2)
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


def test_one_executable_with_every_operator(gpu_client):
    # two attentions of different kernels and a sampler share one workspace, one after the other
    new, lengths = [30, 5], [900, 700]
    module, ins = op.attention_case(new, lengths, 4, 2, 64, 16, "bf16", seed=21)
    step, step_ins = op.attention_case([1] * 3, [500, 70, 600], 4, 2, 64, 16, "bf16", seed=22)
    draw, draw_ins = op.sample_case(np.random.RandomState(23).randn(3, 40000), "f32", 0.9, [0, 50, 0], [1, 1, .9], 0, [.1, .5, .9])
    parts, params, results, n = [], [], [], 0
    for m in (module, step, draw, module):
        head, call = m.split("\n")[1], m.split("\n")[2]
        for ty in [p.split(": ", 1)[1] for p in head[head.index("(") + 1:head.index(") ->")].split(", %")]:
            params.append(ty)
        count = call.count("%arg")
        call = call.replace("%0", f"%r{len(parts)}")
        for i in reversed(range(count)):
            call = call.replace(f"%arg{i},", f"%in{n + i},").replace(f"%arg{i})", f"%in{n + i})")
        n += count
        out = call.rsplit("-> ", 1)[1].strip("() ")
        for i, ty in enumerate(out.split(", ")):
            results.append((f"%r{len(parts)}" + (f"#{i}" if ", " in out else ""), ty))
        parts.append(call)
    text = (f"module {{\n  func.func @main({', '.join(f'%in{i}: {t}' for i, t in enumerate(params))}) -> ({', '.join(t for _, t in results)}) {{\n"
            + "\n".join(parts) + f"\n    return {', '.join(r for r, _ in results)} : {', '.join(t for _, t in results)}\n  }}\n}}\n")
    (a, b, token, _, again), _ = run(gpu_client, text, ins + step_ins + draw_ins + ins, ["bf16", "bf16", "i32", "f32", "bf16"])
    for got, m, i in ((a, module, ins), (b, step, step_ins), (again, module, ins)):
        x = op.values(i)
        close(got, oo.paged_attention(x, op.config_of(m))[0], "bf16", attention_error(x, "bf16"), "shared")
    assert np.array_equal(a, again)
    assert np.array_equal(token, oo.sample(op.values(draw_ins), {})[0])


# ------------------------------------------------------------------------------------------------ sample
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_beyond_the_chunks(gpu_client, dtype):
    r = np.random.RandomState(31)
    check_sample(gpu_client, r.randn(4, 540000) * 2, dtype, temperature=[0.7, 1.0, 0.0, 1.2], top_k=[0, 40, 0, 3000],
                 top_p=[0.9, 1.0, 1.0, 0.8], uniform=[0.3, 0.99, 0.5, 0.7])


@pytest.mark.parametrize("rows, vocab, dtype", [(1, 1, "f32"), (1, 3, "f32"), (1, 3, "bf16"), (1, 7, "f16"), (2, 3, "bf16"), (1, 8, "f16")])
def test_sample_few_bytes(gpu_client, rows, vocab, dtype):
    for u in (0.0, 0.6, 1.0 - 2.0 ** -24):
        check_sample(gpu_client, np.random.RandomState(vocab).randn(rows, vocab), dtype, uniform=u, top_p=0.9, temperature=2.0)


@pytest.mark.parametrize("vocab", [8191, 8193, 16385, 40001, 65537])
def test_sample_at_chunk_borders(gpu_client, vocab):
    r = np.random.RandomState(vocab)
    x = r.randn(6, vocab)
    x[0, :8192] = -np.inf                                             # a chunk without tokens
    x[1, 8190:8194] = np.nan
    x[2, -1] = np.inf
    x[3] = -np.inf
    x[3, [0, vocab - 1]] = [1.0, 1.0]
    x[4] = -np.inf
    for dtype in ("f32", "f16"):                                      # (odd rows of 16 bits begin anywhere)
        check_sample(gpu_client, x, dtype, uniform=r.uniform(0, 1, 6))
        check_sample(gpu_client, x, dtype, uniform=r.uniform(0, 1, 6), top_k=[9, 0, 5, 0, 3, 1500], top_p=[1, .5, 1, .9, .9, .99],
                     min_p=[0, 0, 0, 0, 0, 1e-3])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_large_sets(gpu_client, dtype):
    # more tokens kept than any list holds
    r = np.random.RandomState(32)
    x = r.randn(8, 40000)
    check_sample(gpu_client, x, dtype, top_k=[1023, 1024, 1025, 3000, 20000, 39999, 40000, 2 ** 31 - 1], uniform=r.uniform(0, 1, 8))
    check_sample(gpu_client, x, dtype, temperature=8.0, top_p=[.1, .5, .9, .99, .999, .9999, 1 - 2.0 ** -24, 0.0], uniform=r.uniform(0, 1, 8))
    check_sample(gpu_client, x, dtype, min_p=[1e-9, 1e-6, 1e-4, .01, .3, .9, 1.0, 2.0], uniform=r.uniform(0, 1, 8))


def test_sample_crowded_weights(gpu_client):
    # tens of thousands of weights within an eighth of an octave, or equal, with the border among them
    r = np.random.RandomState(33)
    near = r.randn(6, 30000) * 1e-3
    equal = np.zeros((6, 30000))
    two = np.where(r.rand(6, 30000) < 0.5, 0.0, -1.0)
    for x in (near, equal, two):
        check_sample(gpu_client, x, "f32", top_k=[5000, 1, 17, 4096, 29999, 0], uniform=r.uniform(0, 1, 6))
        check_sample(gpu_client, x, "f32", top_p=[.001, .3, .7, .99, .5, .5], uniform=r.uniform(0, 1, 6))
        check_sample(gpu_client, x, "f32", top_k=[5000, 100, 17, 4096, 29999, 0], top_p=0.7, min_p=0.2, uniform=r.uniform(0, 1, 6))


def test_sample_temperatures(gpu_client):
    r = np.random.RandomState(34)
    x = r.randn(9, 20000) * 3
    t = [1e-38, 1e-6, 1e-3, 0.01, 0.1, 10.0, 1e6, 1e38, np.inf]
    check_sample(gpu_client, x, "f32", temperature=t, uniform=r.uniform(0, 1, 9))
    check_sample(gpu_client, x, "f32", temperature=t, uniform=r.uniform(0, 1, 9), top_p=0.6, top_k=500)


def test_sample_more_rows_than_one_launch_takes(gpu_client):
    r = np.random.RandomState(35)
    few, times, v = 8, 500, 8500
    x, u = r.randn(few, v) * 2, np.float32(r.uniform(0, 1, few))
    k, p = np.array([0, 9, 0, 300, 0, 0, 2000, 0]), np.array([1, 1, .8, .9, .5, 1, 1, .95])
    _, small = op.sample_case(x, "bf16", 0.9, k, p, 0.0, u)
    wt, wl = oo.sample(op.values(small), {})
    module, ins = op.sample_case(np.tile(x, (times, 1)), "bf16", 0.9, np.tile(k, times), np.tile(p, times), 0.0, np.tile(u, times))
    (token, logprob), _ = run(gpu_client, module, ins, ["i32", "f32"])
    assert np.array_equal(token.reshape(times, few), np.tile(wt, (times, 1)))
    assert np.all(np.abs(logprob.reshape(times, few) - wl) <= 2.0 ** -23 * np.abs(wl) + 2.0 ** -30)


# ------------------------------------------------------------------------------------------------ rope_append
@pytest.mark.parametrize("shape", [(3, 3, 1, 16, 16, 16, 1), (40, 8, 2, 32, 32, 16, 3), (40, 8, 2, 32, 16, 16, 3), (5, 6, 2, 128, 96, 8, 1),
                                   (1500, 32, 8, 64, 32, 16, 100), (1300, 40, 4, 128, 128, 64, 21), (300, 5, 1, 256, 64, 16, 20)], ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_append(gpu_client, shape, interleaved, norm):
    for dtype in ("bf16", "f16"):
        module, ins = op.append_case(*shape, dtype, norm=norm, interleaved=interleaved, start=123456, bad_slots=True, seed=sum(shape))
        (q, kc, vc), _ = run(gpu_client, module, ins, [dtype] * 3)
        x = op.values(ins)
        wq, wk, wv = oo.rope_append(x, op.config_of(module))
        big = lambda w: 2.0 ** -19 * np.abs(w).max(axis=-1, keepdims=True)  # noqa: E731
        close(q, wq, dtype, big(wq), "q")
        close(kc, wk, dtype, big(wk), "keys")
        assert np.array_equal(vc, wv)


@pytest.mark.parametrize("d, rot", [(128, 64), (64, 16), (96, 32)])
def test_rope_append_infinities_stay_where_they_are(gpu_client, d, rot):
    # in the part of a head that is not rotated, and in one pair of the rotated part
    module, ins = op.append_case(9, 4, 2, d, rot, 16, 2, "bf16", norm=False, interleaved=False, start=7, seed=3)
    x = op.values(ins)
    x[0][2, 1, rot], x[0][3, 0, d - 1], x[0][4, 2, 3], x[1][5, 1, rot + 1], x[2][6, 0, 0] = np.inf, np.nan, np.inf, -np.inf, np.nan
    for i in range(3):
        ins[i] = op.host(x[i], "bf16")
    (q, kc, vc), _ = run(gpu_client, module, ins, ["bf16"] * 3)
    with np.errstate(invalid="ignore"):
        wq, wk, wv = oo.rope_append(x, op.config_of(module))
    for got, want in ((q, wq), (kc, wk), (vc, wv)):
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
        ok = np.isfinite(want)
        assert np.all(np.abs(got[ok] - want[ok]) <= 2.0 ** -8 * np.abs(want[ok]) + 2.0 ** -16)


# ------------------------------------------------------------------------------------------------ execute_into
def test_execute_into_refuses_what_does_not_fit(gpu_client):
    module, ins = op.sample_case(np.zeros((2, 50)), "f32", 1.0, 0, 1.0, 0.0, 0.5)
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    bufs = device_buffers(gpu_client, ins)
    outs = [gpu_client.uninitialized_buffer(pjrt.BufferType.S32, (2,)), gpu_client.uninitialized_buffer(pjrt.BufferType.F32, (2,))]
    a, b = [span(x) for x in bufs], [span(x) for x in outs]
    for inputs, results in ((a[:-1], b), (a, b[:1]), ([(a[0][0], a[0][1] - 4)] + a[1:], b), (a, [b[0], (b[1][0], 4)])):
        with pytest.raises(pjrt.PjrtError) as e:
            exe.execute_into(inputs, results)
        assert e.value.code == pjrt.ErrorCode.INVALID_ARGUMENT
    exe.execute_into(a, b)
    sync()
    assert np.array_equal(outs[0].to_numpy(), oo.sample(op.values(ins), {})[0])
