"""The decoding operators on the GPU at the edges of their definitions, results written over buffers that hold other values
before. Tolerances as in test_gpu_operators.py."""
import numpy as np
import pytest
import torch  # noqa: F401  (before the plugin: both then use one HIP runtime)

from oracle import operators as oo
from oracle import stablehlo as sh
from ryft_amd import operators, pjrt
from tests import operator_programs as op
from tests.test_gpu_operators import attention_error, check_sample, close, device_buffers, span, sync

pytestmark = pytest.mark.gpu


def run_over(client, module, ins, outs):
    """The results of one execution into buffers that hold 7s before; outs: (shape, dtype)."""
    exe = client.compile(pjrt.Program.mlir(module))
    bufs = device_buffers(client, ins)
    res = device_buffers(client, [op.host(np.full(shape, 7.0), dt) for shape, dt in outs])
    exe.execute_into([span(b) for b in bufs], [span(b) for b in res])
    sync()
    return [sh.from_raw(b.to_numpy().view(np.uint16) if dt == "f16" else b.to_numpy(), dt).reshape(shape)
            for b, (shape, dt) in zip(res, outs)]


# ------------------------------------------------------------------------------------------------ more queries than keys
MORE_QUERIES = {
    "none": dict(new=[200], lengths=[0], heads=(4, 2)),
    "ten": dict(new=[200], lengths=[10], heads=(4, 2)),
    "behind": dict(new=[100, 3, 300, 0, 90], lengths=[150, 3, 0, 9, 20], heads=(4, 2)),
    "window": dict(new=[200, 70], lengths=[10, 100], heads=(4, 1), window=5),
    "capped": dict(new=[200, 70], lengths=[10, 100], heads=(5, 1), softcap=5.0, slopes=True),
    "not_causal": dict(new=[200, 70], lengths=[10, 0], heads=(4, 2), causal=False),
    # tiles alone fill the chip; ranges of keys; more sequences than a wavefront holds
    "many_tiles": dict(new=[20] * 8 + [300], lengths=[20] * 8 + [0], heads=(64, 64)),
    "ranges": dict(new=[200, 40], lengths=[10, 700], heads=(4, 2)),
    "many": dict(new=[30] * 66 + [200], lengths=[5] * 66 + [0], heads=(8, 8)),
}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", MORE_QUERIES)
def test_more_queries_than_keys(gpu_client, name, d, dtype):
    c = dict(MORE_QUERIES[name])
    new, lengths, heads = (c.pop(k) for k in ("new", "lengths", "heads"))
    module, ins = op.attention_case(new, lengths, *heads, d, 16, dtype, seed=len(name) + d, **c)
    (got,) = run_over(gpu_client, module, ins, [(ins[0].dims, dtype)])
    x = op.values(ins)
    want, = oo.paged_attention(x, op.config_of(module))
    close(got, want, dtype, attention_error(x, dtype), name)
    unseen = ~want.any(axis=(1, 2))
    assert unseen.any() and not got[unseen].any()                     # rows that see nothing are exactly zero


# ------------------------------------------------------------------------------------------------ starts that decrease
@pytest.mark.parametrize("starts, sequences", [([0, 4000] * 1053 + [0], 2106), ([0, 9, 3, 12] + [12] * 400, 403)], ids=["long", "short"])
def test_starts_that_decrease_leave_nothing_behind(gpu_client, starts, sequences):
    # a decoding step whose starts name far more rows than there are (the first: so many that a count of their units in 32 bits
    # ends inside a tile of sequence 311): zeros, and the next call on the same executable gives what the one before gave
    tokens, pages, size, per = max(starts), 3, 512, 255
    r = np.random.RandomState(7)
    lengths = r.randint(1, 3000, sequences)
    lengths[311] = size * per - 100
    module = operators.paged_attention_module(tokens=tokens, sequences=sequences, q_heads=32, kv_heads=8, head_dim=64, pages=pages,
                                              page_size=size, pages_per_sequence=per, scale=0.125)
    cache, good = (pages, 8, size, 64), np.maximum(0, np.arange(sequences + 1) - (sequences - min(sequences, tokens)))
    ins = [op.host(r.randn(tokens, 32, 64), "bf16"), op.host(r.randn(*cache), "bf16"), op.host(r.randn(*cache), "bf16"),
           op.host(r.randint(0, pages, (sequences, per)), "i32"), op.host(good, "i32"), op.host(lengths, "i32")]
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    bufs = device_buffers(gpu_client, ins)
    bad = device_buffers(gpu_client, [op.host(starts, "i32"), op.host(np.full(sequences, size * per), "i32")])
    (out,) = device_buffers(gpu_client, [op.host(np.full((tokens, 32, 64), 7.0), "bf16")])

    def execute(args):
        exe.execute_into([span(b) for b in args], [span(out)])
        sync()
        return sh.from_raw(out.to_numpy(), "bf16")

    want = execute(bufs)
    assert np.isfinite(want).all() and want[:min(sequences, tokens)].any() and not want[sequences:].any()
    for _ in range(2):
        assert not execute(bufs[:4] + bad).any()
        assert np.array_equal(execute(bufs), want)


# ------------------------------------------------------------------------------------------------ windows without causality
OPEN_WINDOWS = {
    # a query sees from its window's first key to the sequence's last
    "step": dict(new=[1, 3], lengths=[900, 200], heads=(8, 2, 128)),
    "step_64": dict(new=[1, 3], lengths=[900, 200], heads=(4, 4, 64)),
    "prompt": dict(new=[100, 40], lengths=[100, 200], heads=(4, 2, 128)),
    "ranges": dict(new=[20, 33], lengths=[3000, 700], heads=(4, 1, 64)),
    "many": dict(new=[20] * 66, lengths=[40 + 3 * i for i in range(66)], heads=(8, 8, 64)),
    "any": dict(new=[1, 20], lengths=[300, 90], heads=(4, 2, 80)),
}


@pytest.mark.parametrize("window", [1, 30, 400])
@pytest.mark.parametrize("name", OPEN_WINDOWS)
def test_windows_without_causality(gpu_client, name, window):
    c = dict(OPEN_WINDOWS[name])
    new, lengths, heads = (c.pop(k) for k in ("new", "lengths", "heads"))
    module, ins = op.attention_case(new, lengths, *heads, 16, "bf16", seed=23, window=window, causal=False)
    (got,) = run_over(gpu_client, module, ins, [(ins[0].dims, "bf16")])
    x = op.values(ins)
    want, = oo.paged_attention(x, op.config_of(module))
    close(got, want, "bf16", attention_error(x, "bf16"), name)


# ------------------------------------------------------------------------------------------------ caps of any size
CAPPED = {
    # a decoding step, prompts, ranges of keys, the kernel for any type and head dim
    "step": dict(new=[1, 1, 3], lengths=[300, 40, 70], heads=(8, 2, 128)),
    "step_64": dict(new=[1, 1, 3], lengths=[300, 40, 70], heads=(4, 4, 64), slopes=True),
    "prompt": dict(new=[150, 9], lengths=[150, 64], heads=(4, 2, 128)),
    "prompt_64": dict(new=[150, 9], lengths=[150, 64], heads=(4, 2, 64), slopes=True),
    "ranges": dict(new=[30, 2], lengths=[1500, 700], heads=(4, 1, 64)),
    "any": dict(new=[1, 30], lengths=[200, 90], heads=(4, 2, 80)),
}


@pytest.mark.parametrize("poison", [False, True], ids=["", "poison"])
@pytest.mark.parametrize("softcap", [1e-42, 1e-38, 1e-6, 0.25, 1.0, 1e3, 1e5, 1e6, 1e7, 1e9, 1e20, 1e38, 3.4028234663852886e38], ids=str)
@pytest.mark.parametrize("name", CAPPED)
def test_caps_of_any_size(gpu_client, name, softcap, poison):
    # far above the scores a cap changes nothing, far below them every score is the cap's sign; also beside infinite and
    # NaN keys that nothing sees
    c = dict(CAPPED[name])
    new, lengths, heads = (c.pop(k) for k in ("new", "lengths", "heads"))
    for dtype in ("bf16", "f32") if name == "any" else ("bf16", "f16"):
        module, ins = op.attention_case(new, lengths, *heads, 16, dtype, seed=17, softcap=softcap, poison=poison, **c)
        q = op.values(ins)[0]
        q[-1] = 0.0                                                   # (scores of zero stay so under any cap)
        ins[0] = op.host(q, dtype)
        (got,) = run_over(gpu_client, module, ins, [(ins[0].dims, dtype)])
        x = op.values(ins)
        want, = oo.paged_attention(x, op.config_of(module))
        assert np.isfinite(want).all()
        close(got, want, dtype, attention_error(x, dtype), (name, softcap, dtype))


@pytest.mark.parametrize("softcap", [40.0, 300.0, 500.0, 5000.0], ids=str)
@pytest.mark.parametrize("new, lengths, d", [([1, 2], [300, 70], 128), ([1, 2], [300, 70], 64), ([70], [200], 128), ([70], [200], 64),
                                             ([3], [90], 80)], ids=str)
def test_caps_near_scores_of_hundreds(gpu_client, new, lengths, d, softcap):
    # scores on both sides of half the cap, beside each other in a block; keys past the first of small size, so that scores
    # near zero are weighed against each other while larger ones of either sign stand among them
    hkv, tokens = 2, sum(new)
    module, ins = op.attention_case(new, lengths, 4, hkv, d, 16, "bf16", seed=19, softcap=softcap)
    q, kc = op.values(ins)[:2]
    q[:], kc[:] = np.abs(q), kc * 0.01
    kc[:, :, 3] = -300.0 * np.abs(kc[:, :, 3]) / 0.01 / np.sqrt(d)    # (far below the others, and far past the cap's half)
    ins[0], ins[1] = op.host(q, "bf16"), op.host(kc, "bf16")
    (got,) = run_over(gpu_client, module, ins, [(ins[0].dims, "bf16")])
    x = op.values(ins)
    want, = oo.paged_attention(x, op.config_of(module))
    assert np.isfinite(want).all()
    close(got, want, "bf16", attention_error(x, "bf16"), softcap)


# ------------------------------------------------------------------------------------------------ filters at their ends
@pytest.mark.parametrize("vocab", [40, 9000, 540000])
def test_min_p_above_one_keeps_one_token(gpu_client, vocab):
    # of several largest logits the first, as the largest is always kept and nothing else is; NaN is no bound that any meets
    x = np.random.RandomState(vocab).randn(6, vocab) - 9
    x[:, [7, 11, vocab - 1]] = 2.0
    x[4, 11] = np.inf
    x[5] = np.nan
    for min_p in (1.0 + 2.0 ** -23, 2.0, np.inf, np.nan):
        token = check_sample(gpu_client, x, "f32", min_p=min_p, uniform=[0.0, 0.5, 0.9, 0.99, 0.7, 0.1], top_k=[0, 0, 2, 9, 0, 0],
                             top_p=[1.0, 0.5, 1.0, 0.9, 1.0, 1.0])
        assert list(token) == [7, 7, 7, 7, 11, -1]
    assert len(set(check_sample(gpu_client, x[:3], "f32", min_p=1.0, uniform=[0.1, 0.5, 0.9]))) == 3  # (all three)


@pytest.mark.parametrize("vocab, near", [(5000, 100), (5000, 10), (40000, 3), (540000, 100), (30000, 20000)], ids=str)
def test_uniform_zero_takes_the_first_token_kept(gpu_client, vocab, near):
    # all but `near` tokens weigh so little that no sum over the row shows them, but some are kept: with a uniform number of 0
    # the first of those is the token, and never one that a filter has cut off
    r = np.random.RandomState(vocab + near)
    x = np.full((8, vocab), -80.0) - 20 * r.rand(8, vocab)
    for row in range(8):
        x[row, r.permutation(vocab - 900)[:near] + 900] = r.rand(near) * 1e-3
    x[:, 0] = -101.0                                                  # (the least of all)
    x[1, :800] = -800.0                                               # (no weight at all: 0 in 64 bits)
    token = check_sample(gpu_client, x, "f32", uniform=0.0, top_k=[0, 0, 2000, 4999, 500, 11, 0, 0],
                         min_p=[0, 0, 0, 0, 0, 0, 1e-40, 1e-36], top_p=1.0)
    assert token[0] == 0 and (token[2:] > 0).all()
    check_sample(gpu_client, x, "f32", uniform=0.0, top_k=[0, 0, 2000, 4999, 500, 11, 0, 0], top_p=0.9)
    check_sample(gpu_client, x, "f32", uniform=0.5, top_k=[0, 0, 2000, 4999, 500, 11, 0, 0], min_p=[0, 0, 0, 0, 0, 0, 1e-40, 1e-36])


# ------------------------------------------------------------------------------------------------ chains of appends
CHAINS = {
    "two": dict(steps=2), "three": dict(steps=3), "caches_first": dict(steps=2, returns=["%r1#2", "%r1#1", "%r0#0", "%r1#0"]),
    "between": dict(steps=2, returns=["%r0#1", "%r1#1", "%r1#2"]), "keys_alone": dict(steps=3, returns=["%r2#1"]),
    "not_aliased": dict(steps=2, aliased=False), "same_cache": dict(steps=1, returns=["%r0#1", "%r0#2"]),
}


@pytest.mark.parametrize("donate", [False, True])
@pytest.mark.parametrize("name", CHAINS)
def test_chains_of_appends(gpu_client, name, donate):
    module, ins = op.append_chain(seed=len(name), **CHAINS[name])
    if name == "same_cache":
        c = "tensor<2x2x16x64xbf16>"
        module = module.replace("%kc, %vc)", "%e, %e)").replace("    %r0:3", f"    %e = stablehlo.add %kc, %vc : {c}\n    %r0:3")
    exe = gpu_client.compile(pjrt.Program.mlir(module))
    want = sh.evaluate(module, op.values(ins))
    bufs = device_buffers(gpu_client, ins)
    out = exe.execute([[pjrt.ExecutionInput(b, donatable=donate and i in (1, 2)) for i, b in enumerate(bufs)]])[0]
    out.done.await_()
    for n, (b, (w, _)) in enumerate(zip(out.outputs, want)):
        got = sh.from_raw(b.to_numpy(), "bf16")
        close(got, w, "bf16", 2.0 ** -8 * np.abs(w) + 2.0 ** -18 * np.abs(w).max(), (name, n))  # (the oracle rounds too)
    if not donate:                                                    # the operands are as they were
        for i in (1, 2):
            assert np.array_equal(sh.from_raw(bufs[i].to_numpy(), "bf16"), op.values(ins)[i])
