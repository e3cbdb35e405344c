"""The loss against a teacher's top logits and labels, and its gradient (katsu_cuda_distill_fwd, _bwd)."""
import numpy as np
import pytest

import vocab_ref as ref
from katsu_b200 import cabi
from parity_util import DeviceArrays
from test_block_norm import anywhere  # noqa: F401 (fixture)


def inputs(rows, vocab, top, seed=0, spread=2.0):
    """Lists with duplicates and holes, labels with holes, weights of 0 among others."""
    rng = np.random.default_rng([seed, rows, vocab, top])
    z = (spread * rng.standard_normal((rows, vocab))).astype(np.float32)
    index = rng.integers(0, vocab, (rows, top))
    index[rng.random((rows, top)) < 0.1] = -1
    if top > 2:
        index[::2, 1] = index[::2, 0]
        index[::3, -1] = vocab
    at = np.clip(index, 0, vocab - 1)
    teacher = (np.take_along_axis(z, at, 1) + rng.standard_normal((rows, top))).astype(np.float32)
    labels = ref.zipf(rng, vocab, rows)
    if top:
        labels[::4] = at[::4, 0]
    labels[1::5] = -100
    weight = rng.random(rows).astype(np.float32) + np.float32(0.1)
    weight[2::7] = 0
    g = (rng.random(rows) - 0.3).astype(np.float32)
    return {"z": z, "teacher": teacher, "index": index, "labels": labels, "weight": weight, "g": g}


def run(ctx, a, T=1.0, soft=1.0, hard=0.0, shift=0, out_shift=0, in_place=False, accumulate=None, g=True, loss=True, labels=True, weight=True):
    """(loss of the forward, loss of the backward, gradient)."""
    rows, vocab = a["z"].shape
    top = a["index"].shape[1]
    edge = np.full(4, 7.0, np.float32)
    start = np.full((rows, vocab), np.nan, np.float32) if accumulate is None else accumulate
    with DeviceArrays(ctx, z=np.concatenate([edge[:shift], a["z"].reshape(-1), edge]), t=a["teacher"], i=ref.device_ints(a["index"]),
                      l=ref.device_ints(a["labels"]), w=a["weight"], g=a["g"],
                      d=np.concatenate([edge[:out_shift], start.reshape(-1), edge])) as d:
        d.alloc("fwd", rows, fill=np.nan), d.alloc("bwd", rows, fill=np.nan)
        common = (d["z"] + 4 * shift, d["t"], d["i"], d["l"] if labels else None, d["w"] if weight else None, T, soft, hard)
        ctx.distill_fwd(*common, d["fwd"], rows, vocab, top)
        out, name, at = (common[0], "z", shift) if in_place else (d["d"] + 4 * out_shift, "d", out_shift)
        ctx.distill_bwd(*common, d["g"] if g else None, d["bwd"] if loss else None, out, rows, vocab, top, int(accumulate is not None))
        dz = d.get(name)
        assert (dz[:at] == 7).all() and (dz[at + rows * vocab:] == 7).all()
        if not in_place:
            z = d.get("z")
            assert np.array_equal(z[shift: shift + rows * vocab], a["z"].reshape(-1), equal_nan=True)
        return d.get("fwd"), d.get("bwd"), dz[at: at + rows * vocab].reshape(rows, vocab)


def check(ctx, a, T=1.0, soft=1.0, hard=0.0, labels=True, weight=True, g=True, **more):
    want, off, dz, doff = ref.distill(a["z"], a["teacher"], a["index"], a["labels"] if labels else None, a["weight"] if weight else None,
                                      T, soft, hard, a["g"] if g else None)
    fwd, bwd, got = run(ctx, a, T, soft, hard, labels=labels, weight=weight, g=g, **more)
    ref.assert_near(fwd, want, off, "loss")
    if more.get("loss", True):  # (the two calls cut long rows into different parts: their sums agree to roundings, not bit for bit)
        ref.assert_near(bwd, want, off, "loss beside the gradient")
    if more.get("accumulate") is not None:
        before = more["accumulate"].astype(np.float64)
        # added to twice at listed tokens: the row's part, then the list's
        dz, doff = dz + before, doff + 2 * ref.U * (np.abs(before) + np.abs(dz)) + 2 * ref.U * np.abs(dz + before)
    ref.assert_near(got, dz, doff, "gradient")
    return fwd, got


# vocabularies around what a thread's accesses, a block of 128, 256 and 512 threads, and clusters of two to eight hold
SHAPES = [(1, 1, 1), (3, 2, 1), (5, 7, 7), (9, 33, 40), (4, 128, 3), (33, 1000, 10), (7, 4093, 64), (3, 4094, 64), (5, 8190, 17), (2, 8191, 5),
          (3, 16382, 100), (4, 16384, 9), (3, 32768, 64), (9, 50021, 17), (2, 65537, 33), (2, 131066, 64), (1, 131072, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,soft,hard", [(1.0, 1.0, 0.0), (2.0, 0.5, 0.5), (0.7, 1.0, 0.0), (1.0, 0.6, 0.4), (3.0, 0.0, 1.0)])
@pytest.mark.parametrize("rows,vocab,top", SHAPES)
def test_loss_and_gradient(ctx, rows, vocab, top, T, soft, hard):
    check(ctx, inputs(rows, vocab, top), T, soft, hard)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,top", [(1003, 64), (1003, 1000), (4100, 1024), (40001, 1023), (140000, 1024)])
def test_tokens_listed_many_times(ctx, vocab, top):
    """A row of one token only, of two tokens in turn, of pairs far apart, of pairs next to each other, of few tokens at random, and one
    whose places behind the tenth are filled up with a token at a teacher's logit of -infinity."""
    a = inputs(7, vocab, top, seed=3)
    rng, j = np.random.default_rng(vocab), np.arange(top)
    pairs = rng.permutation(vocab)[:top]
    a["index"] = np.stack([np.full(top, vocab - 1), j % 2, pairs[j % (top // 2)], pairs[j // 2], rng.integers(0, 40, top), np.where(j < 10, j + 5, 7), pairs])
    a["teacher"][5, 10:] = -np.inf
    a["labels"] = np.array([vocab - 1, 1, pairs[0], -1, 7, 7, pairs[-1]])
    a["weight"][:] = 1.5
    listed = np.stack([np.bincount(i, minlength=vocab) for i in a["index"]])
    for T, soft, hard in ((1.0, 1.0, 0.0), (2.0, 0.5, 0.5)):
        want, off, dz, doff = ref.distill(a["z"], a["teacher"], a["index"], a["labels"], a["weight"], T, soft, hard, a["g"])
        # a token's probability is a sum of as many roundings as it is listed times, of at most 1
        doff = doff + np.abs(a["g"] * a["weight"])[:, None] * soft * T * ref.U * listed
        first = run(ctx, a, T, soft, hard)
        ref.assert_near(first[0], want, off, "loss")
        ref.assert_near(first[1], want, off, "loss beside the gradient")
        ref.assert_near(first[2], dz, doff, "gradient")
        for x, y in zip(first, run(ctx, a, T, soft, hard)):
            assert np.array_equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("T,hard", [(1.0, 0.0), (2.0, 0.5)])
@pytest.mark.parametrize("rows,vocab", [(2, 131073), (1, 262150), (1, 400003)])
def test_rows_that_are_read_twice(ctx, rows, vocab, T, hard):
    check(ctx, inputs(rows, vocab, 20), T, 1.0, hard)
    check(ctx, inputs(rows, vocab, 20), T, 1.0, hard, in_place=True, loss=False)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1000, 1003, 40000, 40001])
@pytest.mark.parametrize("shift,out_shift", [(0, 1), (1, 0), (3, 3), (2, 1)])
def test_any_address(ctx, vocab, shift, out_shift):
    check(ctx, inputs(6, vocab, 12), 2.0, 0.5, 0.5, shift=shift, out_shift=out_shift)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [999, 4096, 40001])
def test_in_place_and_added(ctx, vocab):
    a = inputs(7, vocab, 30)
    plain = check(ctx, a, 2.0, 0.5, 0.5)
    for x, y in zip(plain, check(ctx, a, 2.0, 0.5, 0.5, in_place=True)):
        assert np.array_equal(x, y)
    check(ctx, a, 2.0, 0.5, 0.5, accumulate=np.random.default_rng(5).standard_normal((7, vocab)).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("labels,weight,g,loss", [(False, True, True, True), (True, False, False, True), (False, False, False, False)])
def test_parts_that_are_left_out(ctx, labels, weight, g, loss):
    check(ctx, inputs(11, 3001, 9), 1.5, 0.7, 0.3, labels=labels, weight=weight, g=g, loss=loss)


@pytest.mark.gpu
def test_without_a_teacher_or_entries(ctx):
    a = inputs(6, 700, 0)
    check(ctx, a, 2.0, 1.0, 1.0)  # no list at all: labels alone
    a = inputs(6, 700, 5)
    a["index"][:] = -1
    fwd, got = check(ctx, a, 2.0, 1.0, 0.0)
    assert not fwd.any() and not got.any()
    a["teacher"][:], a["index"][:] = -np.inf, 3
    fwd, got = check(ctx, a, 2.0, 1.0, 0.0)
    assert not fwd.any() and not got.any()
    rows, vocab = a["z"].shape
    with DeviceArrays(ctx, z=a["z"], l=ref.device_ints(a["labels"])) as d:
        d.alloc("loss", rows)
        ctx.distill_fwd(d["z"], None, None, d["l"], None, 1.0, 0.0, 1.0, d["loss"], rows, vocab, 5)  # soft is 0: not looked at
        want, off, _, _ = ref.distill(a["z"], a["teacher"], a["index"], a["labels"], None, 1.0, 0.0, 1.0)
        ref.assert_near(d.get("loss"), want, off)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [900, 20000, 70000])
def test_masked_logits(ctx, vocab):
    """-infinity and the lowest number: tokens of probability 0; where the teacher or the label wants one the loss is infinite."""
    a = inputs(8, vocab, 6)
    a["weight"][:] = 1
    rng = np.random.default_rng(1)
    for low, rows in ((-np.inf, slice(0, 4)), (np.finfo(np.float32).min, slice(4, 8))):
        keep = np.take_along_axis(a["z"][rows], np.clip(a["index"][rows], 0, vocab - 1), 1).copy()
        a["z"][rows][rng.random((4, vocab)) < 0.9] = low
        if low == -np.inf:
            continue
        np.put_along_axis(a["z"][rows], np.clip(a["index"][rows], 0, vocab - 1), keep, 1)
    a["z"][0, 0] = 0.5
    a["index"][0], a["labels"][0] = 0, 0        # what is listed is not masked
    a["index"][1], a["z"][1, 1], a["z"][1, 2] = 1, -np.inf, 0.0  # the teacher wants a masked one
    a["labels"][1] = 2
    a["index"][2], a["z"][2, 1], a["z"][2, 2], a["labels"][2] = 1, 0.0, -np.inf, 2  # the label does
    a["index"][3], a["z"][3, 1], a["labels"][3] = 1, 0.0, 1
    a["labels"][4:] = a["index"][4:, 0]
    a["z"][7] = np.finfo(np.float32).min        # a row of the lowest number: all alike
    fwd, _, got = run(ctx, a, 1.0, 0.5, 0.5)
    want, off, dz, doff = ref.distill(a["z"], a["teacher"], a["index"], a["labels"], a["weight"], 1.0, 0.5, 0.5, a["g"])
    assert np.isinf(want[1]) and np.isinf(want[2]) and np.isfinite(want[[0, 3, 4, 5, 6]]).all()
    fine = [0, 1, 2, 3, 4, 5, 6]
    ref.assert_near(fwd[fine], want[fine], np.where(np.isfinite(off), off, 0)[fine])
    ref.assert_near(got, dz, doff)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [900, 20000, 70000, 140000])
def test_infinities_and_nans_stay_in_their_row(ctx, vocab):
    a = inputs(10, vocab, 6)
    a["weight"][:] = 1
    a["labels"][:] = 3
    a["index"][:] = np.arange(6)
    plain = run(ctx, a, 2.0, 0.5, 0.5)
    bad = {1: np.nan, 3: np.inf, 5: -np.inf}
    for row, v in bad.items():
        a["z"][row, :] = -np.inf
        if row != 5:
            a["z"][row, vocab // 2] = v
    a["z"][7] = np.nan
    a["weight"][7] = 0  # is not read
    a["z"][8], a["index"][8], a["labels"][8] = -np.inf, -1, -1  # neither part
    fwd, bwd, got = run(ctx, a, 2.0, 0.5, 0.5)
    for row in bad:
        assert np.isnan(fwd[row]) and np.isnan(bwd[row]) and np.isnan(got[row]).all()
    for row in (7, 8):
        assert fwd[row] == 0 and bwd[row] == 0 and not got[row].any()
    rest = [0, 2, 4, 6, 9]
    assert np.array_equal(fwd[rest], plain[0][rest]) and np.array_equal(got[rest], plain[2][rest])


@pytest.mark.gpu
def test_far_apart_and_large_logits(ctx):
    """Largest values in other warps and blocks than the rest, numbers up to 1e30, temperatures of 0.01 and 1e4."""
    for vocab in (5000, 40000, 140000):
        a = inputs(4, vocab, 8, spread=30.0)
        a["z"][0, vocab - 1] = 300.0
        a["z"][1, 0] = 1e30
        a["index"][1, 0] = 0
        a["z"][2] = -1e30
        a["z"][2, vocab // 3] = -9e29
        a["index"][2, :] = vocab // 3
        at = np.clip(a["index"], 0, vocab - 1)
        a["teacher"] = (np.take_along_axis(a["z"], at, 1) * np.float32(0.5)).astype(np.float32)
        for T in (0.01, 1.0, 1e4):
            want, off, dz, doff = ref.distill(a["z"], a["teacher"], a["index"], a["labels"], a["weight"], T, 1.0, 0.0, a["g"])
            fwd, _, got = run(ctx, a, T)
            ref.assert_near(fwd, want, off), ref.assert_near(got, dz, doff)


@pytest.mark.gpu
def test_against_differences(ctx):
    """The gradient against differences of the loss's formula in 64 bits."""
    a = inputs(6, 40, 5)
    T, soft, hard, h = 1.7, 0.6, 0.4, 1e-5
    _, _, got = run(ctx, a, T, soft, hard)

    def loss(z):
        # (apart from the gradient: its own straightforward form)
        q, s = z / T - np.log(np.exp(z / T).sum(1, keepdims=True)), z - np.log(np.exp(z).sum(1, keepdims=True))
        out = np.zeros(len(z))
        for i in range(len(z)):
            there = ref.valid(a["index"][i], 40)
            p = np.exp(a["teacher"][i][there].astype(np.float64) / T)
            p /= p.sum()
            out[i] = soft * T * T * (p * (np.log(p) - q[i, a["index"][i][there]])).sum()
            if a["labels"][i] >= 0:
                out[i] -= hard * s[i, a["labels"][i]]
        return out * a["weight"].astype(np.float64) * a["g"].astype(np.float64)

    z = a["z"].astype(np.float64)
    for v in range(40):
        step = np.zeros_like(z)
        step[:, v] = h
        slope = (loss(z + step) - loss(z - step)) / (2 * h)
        # differences: h^2 / 6 times a third derivative (below 4 here), and 2^-52 of losses below 60, twice, over 2 h
        assert np.abs(got[:, v] - slope).max() <= 4 * h * h + 120 * 2.0 ** -52 / h + 300 * ref.U


@pytest.mark.gpu
def test_replayed_and_on_other_streams():
    from test_captured_calls import capture

    a, b = inputs(5, 40001, 12, seed=1), inputs(5, 40001, 12, seed=2)
    contexts, results = [cabi.Context(0) for _ in range(2)], []
    try:
        for c in contexts:
            with DeviceArrays(c, z=a["z"], t=a["teacher"], i=ref.device_ints(a["index"]), l=ref.device_ints(a["labels"]), w=a["weight"],
                              g=a["g"]) as d:
                for name in ("d", "e"):
                    d.alloc(name, a["z"].size, fill=np.nan), d.alloc(name + "loss", 5, fill=np.nan)
                call = lambda out: c.distill_bwd(d["z"], d["t"], d["i"], d["l"], d["w"], 2.0, 0.5, 0.5, d["g"], d[out + "loss"],  # noqa: E731
                                                 d[out], 5, 40001, 12)
                replay = capture(c, lambda: call("d"))
                for x in (b, a):
                    c.h2d(d["z"], x["z"]), c.h2d(d["t"], x["teacher"]), c.h2d(d["i"], ref.device_ints(x["index"]))
                    call("e")
                    replay()
                    assert np.array_equal(d.get("d"), d.get("e")) and np.array_equal(d.get("dloss"), d.get("eloss"))
                del replay
                results.append(d.get("d"))
        assert np.array_equal(*results)
    finally:
        for c in contexts:
            c.close()


@pytest.mark.gpu
def test_no_rows(ctx):
    ctx.distill_fwd(None, None, None, None, None, 1.0, 1.0, 1.0, None, 0, 5, 3)
    ctx.distill_bwd(None, None, None, None, None, 1.0, 1.0, 1.0, None, None, None, 0, 0, 0)


NAMES = ["logits", "teacher", "index", "labels", "weight", "temperature", "soft", "hard", "g", "loss", "dlogits", "rows", "vocab", "top", "accumulate"]
FWD = [n for n in NAMES if n not in ("g", "dlogits", "accumulate")]
BASE = {n: 0x100000 + 0x1000 * i for i, n in enumerate(NAMES)}
BASE.update(temperature=2.0, soft=1.0, hard=1.0, rows=4, vocab=8, top=2, accumulate=0)


@pytest.mark.parametrize("why,change", [
    ("below", {"rows": 1 << 31}), ("below", {"vocab": 1 << 31}), ("KATSU_DISTILL_MAX_TOP", {"top": 1025}), ("temperature", {"temperature": 0.0}),
    ("temperature", {"temperature": -1.0}), ("temperature", {"temperature": float("nan")}), ("temperature", {"temperature": float("inf")}),
    ("finite", {"soft": float("inf")}), ("finite", {"hard": float("nan")}), ("vocabulary", {"vocab": 0}), ("logits is null", {"logits": None}),
    ("teacher or index", {"teacher": None}), ("teacher or index", {"index": None}), ("loss is null", {"loss": None}), ("dlogits is null", {"dlogits": None}),
    ("whole element", {"logits": 0x100002}), ("whole element", {"dlogits": 0x900001}), ("whole element", {"labels": 0x900003}),
    ("overlaps", {"loss": BASE["weight"] + 12}), ("overlaps", {"loss": BASE["logits"] + 124}), ("overlaps", {"dlogits": BASE["logits"] + 4}),
    ("overlaps", {"dlogits": BASE["index"] - 124}), ("overlaps", {"dlogits": BASE["g"]}), ("overlaps", {"dlogits": BASE["logits"], "accumulate": 1}),
    ("loss and dlogits", {"dlogits": 0x200000, "loss": 0x20007c}), ("null context", {"ctx": None})])
def test_refusals(anywhere, why, change):  # noqa: F811
    args = {**BASE, **change}
    lib = cabi.load()
    handle = None if "ctx" in change else anywhere
    calls = []
    if not set(change) & {"g", "dlogits", "accumulate"}:
        calls.append(lambda: lib.katsu_cuda_distill_fwd(handle, *(args[n] for n in FWD)))
    if change != {"loss": None}:
        calls.append(lambda: lib.katsu_cuda_distill_bwd(handle, *(args[n] for n in NAMES)))
    for call in calls:
        assert call() == cabi.ERR_INVALID_ARG
        assert why in lib.katsu_cuda_last_error_string().decode()
