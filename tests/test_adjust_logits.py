"""Penalties, biases and masks on the logits of a served model (katsu_cuda_adjust_logits)."""
import numpy as np
import pytest

import vocab_ref as ref
from katsu_b200 import cabi
from parity_util import DeviceArrays
from test_block_norm import anywhere  # noqa: F401 (fixture)

PARTS = ["prompts", "lengths", "repetition", "presence", "frequency", "bias", "allowed"]


def inputs(rows, vocab, cols, biases=0, allowed=None, seed=0):
    rng = np.random.default_rng([seed, rows, vocab, cols, biases])
    a = {"z": (3 * rng.standard_normal((rows, vocab))).astype(np.float32), "history": ref.zipf(rng, vocab, (rows, cols)),
         "lengths": rng.integers(0, cols + 1, rows), "prompts": rng.integers(0, cols + 1, rows),
         "repetition": (1 + 0.3 * rng.random(rows)).astype(np.float32), "presence": rng.standard_normal(rows).astype(np.float32),
         "frequency": (0.5 * rng.random(rows)).astype(np.float32), "bias_tokens": rng.integers(0, vocab, (rows, biases)),
         "bias": (5 * rng.standard_normal((rows, biases))).astype(np.float32) if biases else None, "allowed": None}
    a["history"][rng.random((rows, cols)) < 0.05] = -1
    a["history"][rng.random((rows, cols)) < 0.02] = vocab
    a["lengths"][0], a["prompts"][0] = cols + 5, -3   # beyond the ends
    if rows > 1:
        a["lengths"][1], a["prompts"][1] = -7, cols   # no history
    if rows > 2:
        a["lengths"][2], a["prompts"][2] = cols, cols + 9  # a prompt only
    if biases > 2:
        a["bias_tokens"][:, 1] = a["bias_tokens"][:, 0]
        a["bias_tokens"][::2, 2] = -1
        a["bias_tokens"][1::2, 2] = vocab
        if cols:
            a["bias_tokens"][:, 0] = np.clip(a["history"][:, 0], 0, vocab - 1)  # in the history too
    if allowed is not None:
        a["allowed"] = rng.random((rows, vocab)) < allowed
    return a


def run(ctx, a, shift=0, out_shift=0, in_place=False, without=()):
    rows, vocab = a["z"].shape
    cols, biases = a["history"].shape[1], a["bias_tokens"].shape[1] if a["bias"] is not None and "bias" not in without else 0
    edge = np.full(4, 7.0, np.float32)
    arrays = {n: a[n] for n in ("repetition", "presence", "frequency")}
    arrays.update({n: ref.device_ints(a[n]) for n in ("history", "lengths", "prompts")})
    if biases:
        arrays.update(bias=a["bias"], bias_tokens=ref.device_ints(a["bias_tokens"]))
    if a["allowed"] is not None:
        arrays["allowed"] = ref.device_ints(ref.words_of(a["allowed"]))
    with DeviceArrays(ctx, z=np.concatenate([edge[:shift], a["z"].reshape(-1), edge]),
                      out=np.concatenate([edge[:out_shift], np.full(a["z"].size, np.nan, np.float32), edge]), **arrays) as d:
        at = {n: d.ptr.get(n) if n not in without else None for n in PARTS + ["history", "bias_tokens"]}
        if not biases:
            at["bias_tokens"] = None
        out, name, lead = (d["z"] + 4 * shift, "z", shift) if in_place else (d["out"] + 4 * out_shift, "out", out_shift)
        ctx.adjust_logits(d["z"] + 4 * shift, at["history"] or None, at["prompts"], at["lengths"], at["repetition"], at["presence"], at["frequency"],
                          at["bias_tokens"], at["bias"], at["allowed"], out, rows, vocab, cols, biases)
        got = d.get(name)
        assert (got[:lead] == 7).all() and (got[lead + a["z"].size:] == 7).all()
        if not in_place:
            assert np.array_equal(d.get("z")[shift: shift + a["z"].size], a["z"].reshape(-1), equal_nan=True)
        return got[lead: lead + a["z"].size].reshape(rows, vocab)


def want_of(a, without=()):
    at = {n: None if n in without else a[n] for n in PARTS}
    return ref.adjust(a["z"], a["history"], at["prompts"], at["lengths"], at["repetition"], at["presence"], at["frequency"],
                      a["bias_tokens"], at["bias"], at["allowed"])


def check(ctx, a, without=(), **more):
    want, off = want_of(a, without)
    got = run(ctx, a, without=without, **more)
    ref.assert_near(got, want, off)
    return got


SHAPES = [(1, 1, 1, 0, None), (1, 31, 5, 3, 0.5), (3, 33, 100, 4, 0.1), (2, 1000, 1, 0, None), (5, 4096, 300, 7, 0.05), (4, 8189, 50, 0, None),
          (3, 8190, 257, 5, 0.5), (2, 8192, 1000, 40, None), (7, 8193, 33, 1024, 0.9), (3, 50021, 3000, 16, 0.02), (1, 131072, 20000, 300, 0.001),
          (65, 2000, 64, 3, 1.0), (4, 300, 0, 5, 0.3), (300, 70, 20, 0, 0.5)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,cols,biases,allowed", SHAPES)
def test_everything(ctx, rows, vocab, cols, biases, allowed):
    a = inputs(rows, vocab, cols, biases, allowed)
    plain = check(ctx, a)
    assert np.array_equal(plain, check(ctx, a, in_place=True))


@pytest.mark.gpu
@pytest.mark.parametrize("shift,out_shift", [(1, 0), (0, 2), (3, 3), (2, 1)])
@pytest.mark.parametrize("vocab", [1000, 8190, 20003])
def test_any_address(ctx, vocab, shift, out_shift):
    a = inputs(5, vocab, 200, 6, 0.3)
    assert np.array_equal(check(ctx, a, shift=shift, out_shift=out_shift), check(ctx, a))
    check(ctx, a, shift=shift, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("without", [(p,) for p in PARTS] + [tuple(PARTS[:2]), tuple(PARTS[2:5]), tuple(PARTS)], ids=str)
def test_parts_that_are_left_out(ctx, without):
    check(ctx, inputs(6, 3001, 90, 5, 0.2), without=without)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,biases", [(1003, 5), (1003, 1000), (9000, 1024), (140001, 1021)])
@pytest.mark.parametrize("cols,allowed", [(0, None), (50, 0.7)])
def test_tokens_with_many_biases(ctx, vocab, biases, cols, allowed):
    """A row of one token only, of two in turn, of pairs far apart and of pairs next to each other, of few tokens at random with biases of 0
    among them, and of different tokens."""
    a = inputs(6, vocab, cols, biases, allowed, seed=8)
    rng, j = np.random.default_rng(vocab), np.arange(biases)
    some = np.resize(rng.permutation(vocab), biases)
    a["bias_tokens"] = np.stack([np.full(biases, vocab - 1), j % 2, some[j % (biases // 2)], some[j // 2], rng.integers(0, 40, biases), some])
    a["bias"][4, ::3] = 0.0
    got = check(ctx, a)
    assert np.array_equal(got, check(ctx, a, in_place=True)) and np.array_equal(got, check(ctx, a, shift=3))


@pytest.mark.gpu
def test_untouched_logits_keep_their_bits(ctx):
    bits = np.random.default_rng(4).integers(0, 2 ** 32, (3, 5000), dtype=np.uint32)
    a = inputs(3, 5000, 40, 0, None)
    a["z"] = bits.view(np.float32)
    untouched = np.ones((3, 5000), bool)
    for i in range(3):
        h = a["history"][i]
        untouched[i, h[ref.valid(h, 5000)]] = False
    for in_place in (False, True):
        got = run(ctx, a, in_place=in_place)
        assert np.array_equal(got.view(np.uint32)[untouched], bits[untouched])


@pytest.mark.gpu
def test_infinities_and_nans(ctx):
    """In places that a mask takes away they do not show; elsewhere they are what the formula makes of them."""
    a = inputs(4, 900, 60, 8, 0.5)
    rng = np.random.default_rng(8)
    odd = rng.random(a["z"].shape) < 0.3
    a["z"][odd] = rng.choice([np.nan, np.inf, -np.inf, np.finfo(np.float32).min], odd.sum())
    a["bias"][0, 3], a["bias"][1, 4] = np.inf, np.nan
    a["allowed"][3] = False  # a row without a token
    want, off = want_of(a)
    got = run(ctx, a)
    ref.assert_near(got, want, np.where(np.isfinite(off), off, 0))
    assert (got[~a["allowed"]] == -np.inf).all()


@pytest.mark.gpu
def test_a_token_that_is_everywhere(ctx):
    a = inputs(2, 9000, 40000, 0, None)
    a["history"][:] = 8999
    a["lengths"][:], a["prompts"][:] = 40000, [0, 1]
    got = check(ctx, a)
    assert got[0, 8999] < -1000 or a["frequency"][0] < 0.03


@pytest.mark.gpu
def test_replayed_and_on_other_streams():
    from test_captured_calls import capture

    a, b = inputs(4, 9001, 100, 5, 0.5, seed=1), inputs(4, 9001, 100, 5, 0.5, seed=2)
    contexts, results = [cabi.Context(0) for _ in range(2)], []
    try:
        for c in contexts:
            arrays = {n: a[n] for n in ("z", "repetition", "presence", "frequency", "bias")}
            ints = lambda x: {**{n: ref.device_ints(x[n]) for n in ("history", "lengths", "prompts", "bias_tokens")},  # noqa: E731
                              "allowed": ref.device_ints(ref.words_of(x["allowed"]))}
            with DeviceArrays(c, **arrays, **ints(a)) as d:
                d.alloc("d", a["z"].size), d.alloc("e", a["z"].size)
                call = lambda out: c.adjust_logits(d["z"], d["history"], d["prompts"], d["lengths"], d["repetition"], d["presence"],  # noqa: E731
                                                   d["frequency"], d["bias_tokens"], d["bias"], d["allowed"], d[out], 4, 9001, 100, 5)
                replay = capture(c, lambda: call("d"))
                for x in (b, a):  # the next token's step: other logits, one more token, another state of the grammar
                    c.h2d(d["z"], x["z"])
                    for n, v in ints(x).items():
                        c.h2d(d[n], v)
                    call("e")
                    replay()
                    assert np.array_equal(d.get("d"), d.get("e"))
                    ref.assert_near(d.get("d"), *want_of({**a, **{n: x[n] for n in ("z", "history", "lengths", "prompts", "bias_tokens", "allowed")}}))
                del replay
                results.append(d.get("d"))
        assert np.array_equal(*results)
    finally:
        for c in contexts:
            c.close()


NAMES = ["logits", "history", "prompts", "lengths", "repetition", "presence", "frequency", "bias_tokens", "bias", "allowed", "out", "rows", "vocab",
         "history_cols", "biases"]
BASE = {n: 0x100000 + 0x1000 * i for i, n in enumerate(NAMES)}
BASE.update(rows=4, vocab=8, history_cols=3, biases=2)


@pytest.mark.parametrize("why,change", [
    ("below", {"rows": 1 << 31}), ("below", {"vocab": 1 << 31}), ("below", {"history_cols": 1 << 31}), ("KATSU_LOGITS_MAX_BIASES", {"biases": 1025}),
    ("logits or out", {"logits": None}), ("logits or out", {"out": None}), ("history is null", {"history": None}), ("bias_tokens or bias", {"bias": None}),
    ("bias_tokens or bias", {"bias_tokens": None}), ("whole element", {"logits": 0x100001}), ("whole element", {"out": 0x900002}),
    ("whole element", {"allowed": 0x900002}), ("overlaps", {"out": BASE["logits"] + 4}), ("overlaps", {"out": BASE["history"] + 44}),
    ("overlaps", {"out": BASE["allowed"] - 124}), ("overlaps", {"out": BASE["frequency"] + 12}), ("overlaps", {"out": BASE["bias"] + 28}),
    ("null context", {"ctx": None})])
def test_refusals(anywhere, why, change):  # noqa: F811
    args = {**BASE, **change}
    lib = cabi.load()
    assert lib.katsu_cuda_adjust_logits(None if "ctx" in change else anywhere, *(args[n] for n in NAMES)) == cabi.ERR_INVALID_ARG
    assert why in lib.katsu_cuda_last_error_string().decode()
