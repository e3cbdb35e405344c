"""The norms, the 8-bit product and the clipped step one behind the other over the same buffers, as a training loop calls them:
nothing waits between the calls, and every one reads what those in front of it have just written."""
import numpy as np
import pytest

from parity_util import DeviceArrays
from test_captured_calls import capture
from test_int8 import floats

STEPS = 60


def state(rows, cols):
    rng = np.random.default_rng([rows, cols])
    f = lambda *s, m=0.0, d=1.0: (m + d * rng.standard_normal(s)).astype(np.float32)  # noqa: E731
    return {"x": f(rows, cols), "h": f(rows, cols), "post_w": f(cols, m=1.0, d=0.2), "pre_w": f(cols, m=1.0, d=0.2),
            "w": f(cols, cols, d=cols ** -0.5), "dr": f(rows, cols, d=0.1)}


def run(ctx, a, rows, cols, layer, how):
    with DeviceArrays(ctx, **a) as d:
        for name in ("r", "n", "y", "dx", "dh"):
            d.alloc(name, rows * cols, fill=np.nan)
        for name in ("dpost_w", "dpre_w", "ws"):
            d.alloc(name, cols, fill=np.nan)
        d.alloc("wq", floats(cols, cols)), d.alloc("norm", 1), d.alloc("other", 1)
        eps, kind = 1e-5, int(layer)
        calls = [
            lambda: ctx.int8_quantize_weights(d["w"], d["wq"], d["ws"], cols, cols),
            lambda: ctx.block_norm_fwd(d["x"], d["h"], None, 0, d["post_w"], None, d["pre_w"], None, 0.5, eps, kind, d["r"], d["n"],
                                       rows, cols),
            lambda: ctx.int8_linear(d["n"], d["wq"], d["ws"], None, d["y"], rows, cols, cols),
            lambda: ctx.block_norm_bwd(d["r"], d["h"], None, 0, d["post_w"], None, d["pre_w"], 0.5, eps, kind, d["dr"], d["y"],
                                       d["dx"], d["dh"], None, d["dpost_w"], None, d["dpre_w"], None, rows, cols),
            lambda: ctx.sgd_step_clipped([d["post_w"], d["x"], d["pre_w"]], [d["dpost_w"], d["dx"], d["dpre_w"]],
                                         [cols, rows * cols, cols], 0.1, 1.0, d["norm"]),
            lambda: ctx.clip_grads([d["dh"]], [d["h"]], [rows * cols], 30.0, d["other"]),
        ]
        seen = []

        def step():
            for call in calls:
                call()
                if how == "waiting":
                    ctx.sync()

        if how == "captured":
            step()  # (a workspace of its size before the capture)
            replay = capture(ctx, step)
            for name, v in a.items():
                ctx.h2d(d[name], v)
            for _ in range(STEPS):
                replay()
        else:
            for _ in range(STEPS):
                step()
        ctx.sync()
        for name in ("x", "h", "post_w", "pre_w", "y", "r", "n", "dh", "norm", "other", "ws"):
            seen.append((name, d.get(name)))
        if how == "captured":
            del replay
    return seen


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("rows,cols", [(1, 512), (2, 4096), (8, 520), (40, 1031), (300, 256), (700, 100), (64, 4100), (160, 8300)])
def test_steps_without_waiting(ctx, rows, cols, layer):
    """The same bits whether the host waits behind every call, behind the last one, or replays one captured step."""
    a = state(rows, cols)
    want = run(ctx, a, rows, cols, layer, "waiting")
    for name, v in want:
        assert np.isfinite(v).all(), name
    for how in ("at once", "captured"):
        for (name, v), (_, got) in zip(want, run(ctx, a, rows, cols, layer, how)):
            assert np.array_equal(v, got), (how, name)


@pytest.mark.gpu
def test_two_contexts_at_once():
    """A host thread to a context, both over their own buffers: what one computes does not depend on the other."""
    import threading

    from katsu_b200 import cabi

    sizes = [(8, 520), (300, 256)], [(160, 8300), (1, 512)]
    contexts = [cabi.Context(0) for _ in sizes]
    try:
        alone = [[run(c, state(*s), *s, True, "waiting") for s in pair] for c, pair in zip(contexts, sizes)]
        together = [[], []]

        def drive(i):
            for s in sizes[i]:
                together[i].append(run(contexts[i], state(*s), *s, True, "at once"))

        threads = [threading.Thread(target=drive, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for want, got in zip(alone, together):
            assert len(got) == 2
            for a, b in zip(want, got):
                assert all(np.array_equal(v, w) for (_, v), (_, w) in zip(a, b))
    finally:
        for c in contexts:
            c.close()
