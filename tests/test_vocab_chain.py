"""The two ends of a language model one behind the other over the same buffers, as training and decoding loops call them, and their
launches."""
import numpy as np
import pytest

import vocab_ref as ref
from katsu_b200 import cabi
from parity_util import DeviceArrays
from test_captured_calls import capture
from test_early_launches import early_launches
from test_int8 import floats

STEPS = 20


def training(rng, count, vocab, cols, top):
    z = rng.standard_normal((count, vocab)).astype(np.float32)
    return {"table": rng.standard_normal((vocab, cols)).astype(np.float32), "w": (rng.standard_normal((cols, vocab)) * cols ** -0.5).astype(np.float32),
            "tokens": ref.device_ints(ref.zipf(rng, vocab, count)), "labels": ref.device_ints(ref.zipf(rng, vocab, count)),
            "index": ref.device_ints(rng.integers(0, vocab, (count, top))), "teacher": z[:, :top].copy()}


def run(ctx, a, count, vocab, cols, top, how):
    with DeviceArrays(ctx, **a) as d:
        for name, size in (("x", count * cols), ("logits", count * vocab), ("dx", count * cols), ("dw", cols * vocab), ("loss", count), ("total", 1),
                           ("dtable", vocab * cols), ("norm", 1)):
            d.alloc(name, size, fill=np.nan)
        calls = [
            lambda: ctx.embed_fwd(d["table"], d["tokens"], 2.0, d["x"], count, vocab, cols),
            lambda: ctx.matmul_fwd(d["x"], d["w"], d["logits"], count, cols, vocab),
            # the gradient in the logits' place
            lambda: ctx.distill_bwd(d["logits"], d["teacher"], d["index"], d["labels"], None, 2.0, 0.5, 0.5, None, d["loss"], d["logits"], count,
                                    vocab, top),
            lambda: ctx.matmul_bwd(d["x"], d["w"], d["logits"], d["dx"], d["dw"], count, cols, vocab),
            lambda: ctx.embed_bwd(d["tokens"], d["dx"], 2.0, d["dtable"], count, vocab, cols),
            lambda: ctx.sgd_step_clipped([d["table"], d["w"]], [d["dtable"], d["dw"]], [vocab * cols] * 2, 0.1, 1.0, d["norm"]),
            lambda: ctx.call("katsu_cuda_sum", d["loss"], d["total"], count),
        ]

        def step():
            for call in calls:
                call()
                if how == "waiting":
                    ctx.sync()

        if how == "captured":
            step()
            replay = capture(ctx, step)
            for name in ("table", "w"):
                ctx.h2d(d[name], a[name])
            for _ in range(STEPS):
                replay()
        else:
            for _ in range(STEPS):
                step()
        ctx.sync()
        seen = {name: d.get(name) for name in ("table", "w", "x", "logits", "loss", "total", "norm", "dtable")}
        if how == "captured":
            del replay
    return seen


@pytest.mark.gpu
@pytest.mark.parametrize("count,vocab,cols,top", [(1, 300, 64, 3), (100, 1001, 48, 7), (300, 517, 33, 20), (9000, 400, 20, 4), (40, 40001, 16, 64)])
def test_steps_without_waiting(ctx, count, vocab, cols, top):
    """The same bits whether the host waits behind every call, behind the last one, or replays one captured step."""
    a = training(np.random.default_rng([count, vocab]), count, vocab, cols, top)
    want = run(ctx, a, count, vocab, cols, top, "waiting")
    for name, v in want.items():
        assert np.isfinite(v).all(), name
    for how in ("at once", "captured"):
        got = run(ctx, a, count, vocab, cols, top, how)
        for name, v in want.items():
            assert np.array_equal(v, got[name]), (how, name)


@pytest.mark.gpu
def test_two_contexts_at_once():
    """A host thread to a context: what one computes does not depend on the other."""
    import threading

    sizes = [(300, 517, 33, 20), (9000, 400, 20, 4)]
    inputs = [training(np.random.default_rng(s), *s) for s in sizes]
    contexts = [cabi.Context(0) for _ in sizes]
    try:
        alone = [run(c, a, *s, "waiting") for c, a, s in zip(contexts, inputs, sizes)]
        together = [None, None]

        def drive(i):
            together[i] = run(contexts[i], inputs[i], *sizes[i], "at once")

        threads = [threading.Thread(target=drive, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for want, got in zip(alone, together):
            assert all(np.array_equal(v, got[name]) for name, v in want.items())
    finally:
        for c in contexts:
            c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,k", [(1, 500, 64), (5, 9001, 48)])
def test_decoding_steps(ctx, rows, vocab, k):
    """A served model's loop without a host in between: lookup, head, adjusted logits; each step appends a token that the test chose."""
    rng = np.random.default_rng([rows, vocab])
    w = rng.standard_normal((k, vocab)).astype(np.float32)
    chosen = rng.integers(0, vocab, (STEPS, rows))
    ones, half = np.ones(rows, np.float32), np.full(rows, 0.5, np.float32)
    with DeviceArrays(ctx, w=w, rep=1.5 * ones, pre=half, fre=half, history=ref.device_ints(np.full((rows, STEPS), -1)),
                      lengths=ref.device_ints(np.zeros(rows)), tokens=ref.device_ints(np.zeros(rows))) as d:
        d.alloc("q", floats(vocab, k)), d.alloc("s", vocab), d.alloc("x", rows * k), d.alloc("z", rows * vocab), d.alloc("out", rows * vocab)
        ctx.int8_quantize_weights(d["w"], d["q"], d["s"], k, vocab)

        def step():
            ctx.int8_embed(d["q"], d["s"], d["tokens"], 1.0, d["x"], rows, vocab, k)
            ctx.int8_linear(d["x"], d["q"], d["s"], None, d["z"], rows, k, vocab)
            ctx.adjust_logits(d["z"], d["history"], None, d["lengths"], d["rep"], d["pre"], d["fre"], None, None, None, d["out"], rows, vocab, STEPS, 0)

        step()
        replay = capture(ctx, step)
        for n in range(STEPS):
            history = np.full((rows, STEPS), -1)
            history[:, :n] = chosen[:n].T
            ctx.h2d(d["history"], ref.device_ints(history)), ctx.h2d(d["lengths"], ref.device_ints(np.full(rows, n)))
            ctx.h2d(d["tokens"], ref.device_ints(chosen[n]))
            replay()
            z = d.get("z").reshape(rows, vocab)
            assert np.isfinite(z).all()
            ref.assert_near(d.get("out"), *ref.adjust(z, history, None, np.full(rows, n), 1.5 * ones, half, half, np.zeros((rows, 0)), None, None))
        del replay


def embed(count, vocab, cols, accumulate):
    def calls(ctx, a):
        table, tokens, y = a(vocab * cols), a(count), a(count * cols)
        ctx.embed_fwd(table, tokens, 1.0, y, count, vocab, cols)
        ctx.embed_bwd(tokens, y, 1.0, table, count, vocab, cols, accumulate)
    return calls


def int8_embed(count, vocab, cols):
    def calls(ctx, a):
        buffers = a(floats(vocab, cols)), a(vocab), a(count), 1.0, a(count * cols)
        for _ in range(2):  # (what starts early has a launch in front)
            ctx.int8_embed(*buffers, count, vocab, cols)
    return calls


def distill(rows, vocab, top):
    def calls(ctx, a):
        z, t, i, loss, dz = a(rows * vocab), a(rows * top), a(rows * top), a(rows), a(rows * vocab)
        ctx.distill_fwd(z, t, i, i, None, 2.0, 0.5, 0.5, loss, rows, vocab, top)
        ctx.distill_bwd(z, t, i, i, None, 2.0, 0.5, 0.5, None, loss, dz, rows, vocab, top)
    return calls


def adjust(rows, vocab, cols):
    def calls(ctx, a):
        z, h, out = a(rows * vocab), a(rows * cols), a(rows * vocab)
        for _ in range(2):
            ctx.adjust_logits(z, h, None, None, None, None, None, None, None, None, out, rows, vocab, cols, 0)
    return calls


# (the buffers hold zeros: token 0 everywhere)
CALLS = {
    "lookup 1 x 4096": embed(1, 100, 4096, 1), "lookup 64 x 1001": embed(64, 100, 1001, 0), "lookup 300 x 4096": embed(300, 100, 4096, 1),
    "lookup 3001 x 515": embed(3001, 2000, 515, 1), "lookup 8192 x 64": embed(8192, 50000, 64, 0), "lookup 20000 x 24": embed(20000, 3000, 24, 0),
    "lookup 300000 x 4": embed(300000, 70000, 4, 1), "lookup 262144 x 16": embed(262144, 1 << 21, 16, 1), "lookup 40000 x 1024": embed(40000, 900, 1024, 0),
    "8 bits 1 x 4096": int8_embed(1, 100, 4096), "8 bits 3000 x 333": int8_embed(3000, 100, 333), "loss 1 x 32768": distill(1, 32768, 64),
    "loss 300 x 1000": distill(300, 1000, 9), "loss 40 x 140000": distill(40, 140000, 64), "logits 1 x 32768": adjust(1, 32768, 100),
    "logits 70 x 50000": adjust(70, 50000, 40000), "logits 2000 x 3000": adjust(2000, 3000, 5),
}


@pytest.mark.gpu
@pytest.mark.parametrize("which", CALLS)
def test_all_blocks_of_early_launches_are_resident_at_once(which):
    ctx, buffers = cabi.Context(0), []

    def allocate(count):
        buffers.append(ctx.alloc(count))
        return buffers[-1]

    try:
        CALLS[which](ctx, allocate)  # (buffers, and a workspace of its size: the capture allocates nothing)
        ctx.sync()
        again = iter(buffers)
        found = early_launches(ctx, lambda: CALLS[which](ctx, lambda count: next(again)))
        assert [launch for launch in found if launch[1] > launch[2]] == []
        for pointer in buffers:
            ctx.free(pointer)
    finally:
        ctx.close()
