"""The norms around a block (katsu_cuda_block_norm_fwd / _bwd) against their formulas in 64 bits, and against differences."""
import itertools

import numpy as np
import pytest

import block_ref
from katsu_b200 import cabi
from parity_util import DeviceArrays, rel_l2

U = 2.0 ** -24  # half a step of f32, relative

WEIGHTS = ("post_w", "post_b", "pre_w", "pre_b")
OUTS = ("dx", "dh", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b")


def tolerance(cols, rows=1):
    """Relative to the 2-norm.  A value goes through fewer than 30 roundings outside the sums; a sum of n terms, taken by up to
    1024 threads and a tree, is off by at most (n / 32 + 15) half steps of the sum of magnitudes, which for these inputs is
    below 2 sqrt(n) times the sums that matter only where they nearly vanish: n / 32 covers that.  The statistics (sums of
    squares, no cancellation) and the two means of the backward enter once each; sums over rows are folded in at most
    rows / 32 + 40 steps."""
    return U * (30 + 3 * (cols / 32 + 15) + (rows / 32 + 40))


def inputs(rows, cols, gate_rows=0, post=True, h=True, pre=True, bias=False, seed=0, spread=1.0, mean=0.0):
    rng = np.random.default_rng([seed, rows, cols, gate_rows])
    f = lambda *s, m=0.0, d=1.0: (m + d * rng.standard_normal(s)).astype(np.float32)  # noqa: E731
    a = {"x": f(rows, cols, m=mean, d=spread), "h": f(rows, cols, m=mean / 2, d=spread) if h else None,
         "gate": f(gate_rows, cols, m=1.0, d=0.3) if gate_rows else None}
    for name, here in (("post", post and h), ("pre", pre)):
        a[name + "_w"] = f(cols, m=1.0, d=0.2) if here else None
        a[name + "_b"] = f(cols, d=0.2) if here and bias else None
    a["dr"], a["dn"] = f(rows, cols), f(rows, cols) if pre else None
    return a


def uploaded(ctx, a, shift=0):
    """The arrays, each `shift` floats behind the start of its allocation."""
    return DeviceArrays(ctx, **{k: np.concatenate([np.zeros(shift, np.float32), v.reshape(-1)]) for k, v in a.items() if v is not None})


def fwd(ctx, d, a, shape, scale, eps, layer, r, n, shift=0):
    p = lambda name: d[name] + 4 * shift if a[name] is not None else None  # noqa: E731
    gate_rows = a["gate"].shape[0] if a["gate"] is not None else 0
    ctx.block_norm_fwd(p("x"), p("h"), p("gate"), gate_rows, *(p(w) for w in WEIGHTS), scale, eps, int(layer), r, n, *shape)


def bwd(ctx, d, a, shape, scale, eps, layer, outs, accumulate=0, shift=0, dr=True):
    p = lambda name: d[name] + 4 * shift if a.get(name) is not None else None  # noqa: E731
    gate_rows = a["gate"].shape[0] if a["gate"] is not None else 0
    ctx.block_norm_bwd(p("r"), p("h"), p("gate"), gate_rows, p("post_w"), p("post_b"), p("pre_w"), scale, eps, int(layer),
                       p("dr") if dr else None, p("dn"), *(outs.get(o) for o in OUTS), *shape, accumulate)


SHAPES = [(1, 1), (1, 4096), (3, 2), (5, 33), (2, 255), (7, 256), (4, 1024), (6, 1367), (3, 4096), (2, 5120), (3, 8191),
          (2, 8192), (2, 16388), (1, 40001), (300, 64), (1022, 96), (900, 4), (2500, 7),
          (1200, 250), (600, 128), (40, 8200), (400, 8452)]


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(ctx, rows, cols, layer):
    a = inputs(rows, cols, gate_rows=1, bias=layer)
    r64, n64 = block_ref.forward(*(a[k] for k in ("x", "h", "gate", *WEIGHTS)), 0.5, 1e-5, layer)
    with uploaded(ctx, a) as d:
        d.alloc("r", rows * cols, fill=np.nan), d.alloc("n", rows * cols, fill=np.nan)
        fwd(ctx, d, a, (rows, cols), 0.5, 1e-5, layer, d["r"], d["n"])
        r, n = d.get("r").reshape(rows, cols), d.get("n").reshape(rows, cols)
    # cols of 1 and 2 make differences from the mean that cancel: the norm of such a row is held to the row's own size
    assert rel_l2(r, r64) <= tolerance(cols)
    np.testing.assert_allclose(n, n64, rtol=0, atol=tolerance(cols) * 60 * np.abs(n64).max() if cols < 32 else 40 * tolerance(cols))
    if cols >= 32:
        assert rel_l2(n, n64) <= tolerance(cols)


def check_backward(got, want, rows, cols, what=""):
    for name, v in got.items():
        w = want[name].reshape(-1)
        if not np.any(w):
            assert not np.any(v), (what, name)
            continue
        assert rel_l2(v, w) <= tolerance(cols, rows), (what, name, rel_l2(v, w))


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("rows,cols", [s for s in SHAPES if s[1] >= 32])
def test_backward(ctx, rows, cols, layer):
    a = inputs(rows, cols, gate_rows=1, bias=layer)
    a["r"] = a.pop("x")
    args = [a[k] for k in ("r", "h", "gate", "post_w", "post_b", "pre_w")]
    want = block_ref.backward(*args, 0.5, 1e-5, layer, a["dr"], a["dn"])
    names = [o for o in OUTS if layer or not o.endswith("_b")]
    with uploaded(ctx, a) as d:
        for o in names:
            d.alloc(o, want[o].size, fill=np.nan)
        bwd(ctx, d, a, (rows, cols), 0.5, 1e-5, layer, {o: d[o] for o in names})
        got = {o: d.get(o) for o in names}
    check_backward(got, want, rows, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("h,post,pre,gate_rows", [p for p in itertools.product([True, False], [True, False], [True, False], [0, 1, 3, 6, 12, 24])
                                                  if (p[0] or not (p[1] or p[3])) and (p[0] or p[2])])
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("cols", [36, 45, 520, 4097])
def test_parts(ctx, h, post, pre, gate_rows, layer, cols):
    """Every part left out, every kind of gate, and outputs left out and added to."""
    rows, scale, eps = 24, -1.25, 1e-6
    a = inputs(rows, cols, gate_rows, post, h, pre, bias=layer, seed=2)
    r64, n64 = block_ref.forward(*(a[k] for k in ("x", "h", "gate", *WEIGHTS)), scale, eps, layer)
    with uploaded(ctx, a) as d:
        outs = {}
        for o, here in (("r", h), ("n", pre)):
            outs[o] = d.alloc("out_" + o, rows * cols, fill=np.nan) if here else None
        fwd(ctx, d, a, (rows, cols), scale, eps, layer, outs["r"], outs["n"])
        if h:
            assert rel_l2(d.get("out_r"), r64) <= tolerance(cols)
        if pre:
            assert rel_l2(d.get("out_n"), n64) <= tolerance(cols)
    a["r"] = a.pop("x")
    args = [a[k] for k in ("r", "h", "gate", "post_w", "post_b", "pre_w")]
    want = block_ref.backward(*args, scale, eps, layer, a["dr"], a["dn"])
    without_dr = block_ref.backward(*args, scale, eps, layer, None, a["dn"])
    names = [o for o in OUTS if o in want and (layer or not o.endswith("_b"))]
    with uploaded(ctx, a) as d:
        for o in names:
            d.alloc(o, want[o].size, fill=np.nan)
        bwd(ctx, d, a, (rows, cols), scale, eps, layer, {o: d[o] for o in names})
        got = {o: d.get(o) for o in names}
        check_backward(got, want, rows, cols)
        # added to what is there: one rounding more
        for o in names:
            d.ctx.h2d(d[o], np.full(want[o].size, 2.0, np.float32))
        bits = sum(getattr(cabi, "BLOCK_" + o.upper()) for o in names)
        bwd(ctx, d, a, (rows, cols), scale, eps, layer, {o: d[o] for o in names}, accumulate=bits)
        for o in names:
            assert rel_l2(d.get(o), 2.0 + want[o]) <= tolerance(cols, rows) + U, o
        # each output alone, and no gradient of r
        for o in names:
            d.ctx.h2d(d[o], np.full(want[o].size, np.nan, np.float32))
            bwd(ctx, d, a, (rows, cols), scale, eps, layer, {o: d[o]})
            assert np.array_equal(d.get(o), got[o]), o
        if pre:
            for o in names:
                d.ctx.h2d(d[o], np.full(want[o].size, np.nan, np.float32))
            bwd(ctx, d, a, (rows, cols), scale, eps, layer, {o: d[o] for o in names}, dr=False)
            check_backward({o: d.get(o) for o in names}, without_dr, rows, cols, "no dr")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,gate_rows", [(640, 128, 1), (640, 128, 2), (640, 128, 640), (2400, 40, 600), (2400, 40, 1200), (6000, 36, 3000)])
def test_many_rows_and_gates(ctx, rows, cols, gate_rows):
    """More rows than blocks: gates of one row for all, of long runs (cut into blocks), of short ones (several to a block)."""
    a = inputs(rows, cols, gate_rows, bias=True, seed=3)
    a["r"] = a.pop("x")
    want = block_ref.backward(*[a[k] for k in ("r", "h", "gate", "post_w", "post_b", "pre_w")], 1.0, 1e-5, True, a["dr"], a["dn"])
    with uploaded(ctx, a) as d:
        for o in OUTS:
            d.alloc(o, want[o].size, fill=np.nan)
        bwd(ctx, d, a, (rows, cols), 1.0, 1e-5, True, {o: d[o] for o in OUTS})
        got = {o: d.get(o) for o in OUTS}
        check_backward(got, want, rows, cols)
        bwd(ctx, d, a, (rows, cols), 1.0, 1e-5, True, {o: d[o] for o in OUTS})
        for o in OUTS:
            assert np.array_equal(d.get(o), got[o]), o  # the same bits again


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("rows,cols", [(400, 5004), (400, 5120), (160, 9000), (160, 12288), (120, 16384)])
def test_rows_wider_than_a_block(ctx, rows, cols, layer):
    """Several rows to each cluster of blocks.  Along a row the values climb by three spreads and more, so that the blocks'
    own means lie far from the row's: differences from it carry that much more of the values' roundings, a factor of 4."""
    a = inputs(rows, cols, gate_rows=2, bias=layer, seed=10)
    climb = np.linspace(-3, 3, cols, dtype=np.float32)
    a["r"], a["h"] = a.pop("x") + climb, a["h"] - climb
    want = block_ref.backward(*[a[k] for k in ("r", "h", "gate", "post_w", "post_b", "pre_w")], 0.5, 1e-5, layer, a["dr"], a["dn"])
    names = [o for o in OUTS if layer or not o.endswith("_b")]
    with uploaded(ctx, a) as d:
        for o in names:
            d.alloc(o, want[o].size, fill=np.nan)
        bwd(ctx, d, a, (rows, cols), 0.5, 1e-5, layer, {o: d[o] for o in names})
        got = {o: d.get(o) for o in names}
        for o in names:
            assert rel_l2(got[o], want[o].reshape(-1)) <= 4 * tolerance(cols, rows), (o, rel_l2(got[o], want[o].reshape(-1)))
        for _ in range(3):  # the same bits again
            bwd(ctx, d, a, (rows, cols), 0.5, 1e-5, layer, {o: d[o] for o in names})
        for o in names:
            assert np.array_equal(d.get(o), got[o]), o


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("cols", [64, 1024, 4096, 8192])
def test_unaligned(ctx, cols, shift):
    rows = 5
    a = inputs(rows, cols, gate_rows=5, bias=True, seed=4)
    r64, n64 = block_ref.forward(*(a[k] for k in ("x", "h", "gate", *WEIGHTS)), 1.0, 1e-6, True)
    want = block_ref.backward(a["x"], *[a[k] for k in ("h", "gate", "post_w", "post_b", "pre_w")], 1.0, 1e-6, True, a["dr"], a["dn"])
    a["r"] = a["x"]
    with uploaded(ctx, a, shift) as d:
        for o, size in [("out_r", rows * cols), ("out_n", rows * cols)] + [(o, want[o].size) for o in OUTS]:
            d.alloc(o, size + 8, fill=7.0)
        fwd(ctx, d, a, (rows, cols), 1.0, 1e-6, True, d["out_r"] + 4 * shift, d["out_n"] + 4 * shift, shift)
        bwd(ctx, d, a, (rows, cols), 1.0, 1e-6, True, {o: d[o] + 4 * shift for o in OUTS}, shift=shift)
        for o, w in (("out_r", r64), ("out_n", n64), *want.items()):
            got = d.get(o)
            assert (got[:shift] == 7).all() and (got[shift + w.size:] == 7).all(), o
            assert rel_l2(got[shift:shift + w.size], w) <= tolerance(cols, rows), o


@pytest.mark.gpu
def test_rows_do_not_touch_each_other(ctx):
    """Infinities, NaNs and rows of zeros stay in their rows; a mean far above the spread keeps its bits; no rows at all."""
    rows, cols = 9, 260
    a = inputs(rows, cols, bias=True, seed=5)
    clean = {k: None if v is None else v.copy() for k, v in a.items()}
    a["h"][2, 7], a["h"][4, 0], a["x"][6, 3] = np.inf, np.nan, -np.inf
    a["h"][1], a["x"][1] = 0.0, 0.0
    for arrays, bad in ((clean, []), (a, [2, 4, 6])):
        r64, n64 = block_ref.forward(*(clean[k] for k in ("x", "h", "gate", *WEIGHTS)), 1.0, 1e-6, True)
        with uploaded(ctx, arrays) as d:
            d.alloc("r", rows * cols, fill=5.0), d.alloc("n", rows * cols, fill=5.0)
            fwd(ctx, d, arrays, (0, cols), 1.0, 1e-6, True, d["r"], d["n"])
            assert (d.get("r") == 5).all() and (d.get("n") == 5).all()
            fwd(ctx, d, arrays, (rows, cols), 1.0, 1e-6, True, d["r"], d["n"])
            n = d.get("n").reshape(rows, cols)
        for i in range(rows):
            if i in bad:
                assert np.isnan(n[i]).any()
            elif i == 1 and bad:  # x = h = 0: the biases alone reach the sum, and its norm is finite
                assert np.isfinite(n[i]).all()
            else:
                assert rel_l2(n[i], n64[i]) <= tolerance(cols), i


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [512, 4096, 9000])
def test_mean_far_above_the_spread(ctx, cols):
    """mean = 1000 spreads: differences from the mean are exact to 2^-24 of the mean, 1000 half steps of the spread, plus what
    the mean itself is off by."""
    a = inputs(4, cols, h=False, post=False, bias=True, seed=6, mean=1000.0)
    _, n64 = block_ref.forward(*(a[k] for k in ("x", "h", "gate", *WEIGHTS)), 1.0, 1e-6, True)
    with uploaded(ctx, a) as d:
        d.alloc("n", 4 * cols, fill=np.nan)
        fwd(ctx, d, a, (4, cols), 1.0, 1e-6, True, None, d["n"])
        assert rel_l2(d.get("n"), n64) <= 1000 * tolerance(cols)


@pytest.mark.gpu
def test_against_differences(ctx):
    """The gradient of sum(dr r + dn n) along random directions, by central differences of the formula in 64 bits."""
    rows, cols, scale, eps = 6, 40, 0.75, 1e-3
    a = inputs(rows, cols, gate_rows=2, bias=True, seed=7)
    names = ("x", "h", "gate", *WEIGHTS)
    for layer in (False, True):
        r64, _ = block_ref.forward(*(a[k] for k in names), scale, eps, layer)
        b = dict(a, r=r64.astype(np.float32))
        outs = dict(zip(names, ("dx", "dh", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b")))
        with uploaded(ctx, b) as d:
            for o in OUTS:
                d.alloc(o, 0 or a[[k for k in names if outs[k] == o][0]].size, fill=np.nan)
            bwd(ctx, d, b, (rows, cols), scale, eps, layer, {o: d[o] for o in OUTS})
            grads = {k: d.get(outs[k]).reshape(a[k].shape).astype(np.float64) for k in names}
        rng = np.random.default_rng(8)
        for k in names:
            way, step = rng.standard_normal(a[k].shape), 1e-4

            def value(t):
                moved = {q: a[q].astype(np.float64) + (t * way if q == k else 0) for q in names}
                r, n = block_ref.forward(*(moved[q] for q in names), scale, eps, layer)
                return (a["dr"] * r).sum() + (a["dn"] * n).sum()

            slope = (value(step) - value(-step)) / (2 * step)
            # differences: step^2 times a third derivative of a few thousand; gradients: f32 sums of up to 240 terms
            assert abs((grads[k] * way).sum() - slope) <= 1e-4 * (np.abs(grads[k] * way).sum() + 1), k


@pytest.mark.gpu
def test_replayed_and_on_other_streams(ctx):
    from test_captured_calls import capture

    rows, cols = 600, 1024
    a = inputs(rows, cols, gate_rows=3, seed=9)
    a["r"] = a["x"]
    names = [o for o in OUTS if not o.endswith("_b")]
    contexts = [cabi.Context(0) for _ in range(2)]
    try:
        results = []
        for c in contexts:
            with uploaded(c, a) as d:
                for o in names:
                    d.alloc(o, a[{"dx": "x", "dh": "h", "dgate": "gate"}.get(o, "pre_w")].size, fill=np.nan)
                call = lambda: bwd(c, d, a, (rows, cols), 1.0, 1e-6, False, {o: d[o] for o in names})  # noqa: E731
                call()
                eager = {o: d.get(o) for o in names}
                replay = capture(c, call)
                for o in names:
                    c.h2d(d[o], np.zeros(eager[o].size, np.float32))
                c.sync()
                replay()
                for o in names:
                    assert np.array_equal(d.get(o), eager[o]), o
                del replay
                results.append(eager)
        for o in names:
            assert np.array_equal(results[0][o], results[1][o])
    finally:
        for c in contexts:
            c.close()


@pytest.fixture
def anywhere():
    """A context where there is a GPU; elsewhere a place that a refused call never looks at."""
    import ctypes

    count = ctypes.c_int32(0)
    if cabi.load().katsu_cuda_device_count(ctypes.byref(count)) == cabi.OK and count.value:
        context = cabi.Context(0)
        yield context.handle
        context.close()
    else:
        yield ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p)


A, B, C, D = 0x10000, 0x20000, 0x30000, 0x40000  # addresses that nothing reads


@pytest.mark.parametrize("why,args", [
    ("kind", (A, B, None, 0, C, None, None, None, 1.0, 1e-6, 2, D, None, 4, 4)),
    ("eps", (A, B, None, 0, C, None, None, None, 1.0, -1.0, 0, D, None, 4, 4)),
    ("eps", (A, B, None, 0, C, None, None, None, 1.0, float("nan"), 0, D, None, 4, 4)),
    ("eps", (A, B, None, 0, C, None, None, None, 1.0, float("inf"), 0, D, None, 4, 4)),
    ("values", (A, B, None, 0, C, None, None, None, 1.0, 1e-6, 0, D, None, 4, 0)),
    ("values", (A, B, None, 0, C, None, None, None, 1.0, 1e-6, 0, D, None, 4, 1 << 30)),
    ("rows", (A, B, None, 0, C, None, None, None, 1.0, 1e-6, 0, D, None, 1 << 61, 4)),
    ("gate", (A, B, None, 1, C, None, None, None, 1.0, 1e-6, 0, D, None, 4, 4)),
    ("gate", (A, B, C, 0, C, None, None, None, 1.0, 1e-6, 0, D, None, 4, 4)),
    ("divide", (A, B, C, 3, C, None, None, None, 1.0, 1e-6, 0, D, None, 4, 4)),
    ("without h", (A, None, C, 1, None, None, A, None, 1.0, 1e-6, 0, None, D, 4, 4)),
    ("without h", (A, None, None, 0, C, None, A, None, 1.0, 1e-6, 0, None, D, 4, 4)),
    ("bias", (A, B, None, 0, None, C, None, None, 1.0, 1e-6, 0, D, None, 4, 4)),
    ("bias", (A, B, None, 0, None, None, None, C, 1.0, 1e-6, 0, D, None, 4, 4)),
    ("n and pre_w", (A, B, None, 0, C, None, C, None, 1.0, 1e-6, 0, D, None, 4, 4)),
    ("n and pre_w", (A, B, None, 0, C, None, None, None, 1.0, 1e-6, 0, D, C, 4, 4)),
    ("nothing", (A, None, None, 0, None, None, None, None, 1.0, 1e-6, 0, None, None, 4, 4)),
    ("nothing", (A, B, None, 0, C, None, A, None, 1.0, 1e-6, 0, None, D, 4, 4)),
    ("x is null", (None, B, None, 0, C, None, None, None, 1.0, 1e-6, 0, D, None, 4, 4)),
    ("output is an input", (A, B, None, 0, C, None, None, None, 1.0, 1e-6, 0, A, None, 4, 4)),
    ("same buffer", (A, B, None, 0, None, None, C, None, 1.0, 1e-6, 0, D, D, 4, 4)),
])
def test_forward_refuses(anywhere, why, args):
    lib = cabi.load()
    assert lib.katsu_cuda_block_norm_fwd(anywhere, *args) == cabi.ERR_INVALID_ARG
    assert why in lib.katsu_cuda_last_error_string().decode()


@pytest.mark.parametrize("why,change", [
    ("accumulate", {"accumulate": 128}), ("accumulate", {"accumulate": -1}), ("without h", {"h": None}),
    ("post_w", {"post_w": None}), ("gate", {"gate": None}), ("gate", {"gate": None, "gate_rows": 0}), ("dn and pre_w", {"dn": None}),
    ("dn and pre_w", {"pre_w": None}), ("r is null", {"r": None}), ("two outputs", {"dx": 0x900, "dh": 0x900}),
    ("output is an input", {"dx": 0x4000}), ("divide", {"gate_rows": 3}), ("kind", {"kind": 7}), ("null context", {"ctx": None})])
def test_backward_refuses(anywhere, why, change):
    names = ["r", "h", "gate", "gate_rows", "post_w", "post_b", "pre_w", "scale", "eps", "kind", "dr", "dn", "dx", "dh", "dgate",
             "dpost_w", "dpost_b", "dpre_w", "dpre_b", "rows", "cols", "accumulate"]
    args = {n: 0x1000 * (i + 1) for i, n in enumerate(names)}
    args.update(r=0x4000, gate_rows=2, scale=1.0, eps=1e-6, kind=1, rows=4, cols=4, accumulate=0)
    args["gate_rows"] = 2
    args.update({k: v for k, v in change.items() if k != "ctx"})
    lib = cabi.load()
    handle = None if "ctx" in change else anywhere
    assert lib.katsu_cuda_block_norm_bwd(handle, *(args[n] for n in names)) == cabi.ERR_INVALID_ARG
    assert why in lib.katsu_cuda_last_error_string().decode()


# rows = 4, cols = 8: x, h, r, n and their gradients 128 bytes, weights 32, a gate of two rows 64
@pytest.mark.parametrize("why,args", [
    ("output is an input", (A, B, None, 0, C, None, None, None, 1.0, 1e-6, 0, A + 124, None, 4, 8)),
    ("output is an input", (A, B, None, 0, C, None, None, None, 1.0, 1e-6, 0, B - 124, None, 4, 8)),
    ("output is an input", (A, B, None, 0, C, None, None, None, 1.0, 1e-6, 0, C + 28, None, 4, 8)),
    ("output is an input", (A, B, C, 2, None, None, A, None, 1.0, 1e-6, 0, D, C + 60, 4, 8)),
    ("output is an input", (A, None, None, 0, None, None, C, B, 1.0, 1e-6, 0, None, B - 124, 4, 8)),
    ("same buffer", (A, B, None, 0, None, None, C, None, 1.0, 1e-6, 0, D, D + 124, 4, 8)),
    ("same buffer", (A, B, None, 0, None, None, C, None, 1.0, 1e-6, 0, D, D - 124, 4, 8)),
])
def test_forward_refuses_overlaps(anywhere, why, args):
    lib = cabi.load()
    assert lib.katsu_cuda_block_norm_fwd(anywhere, *args) == cabi.ERR_INVALID_ARG
    assert why in lib.katsu_cuda_last_error_string().decode()


@pytest.mark.parametrize("why,change", [
    ("two outputs", {"dx": 0x9000, "dh": 0x907c}), ("two outputs", {"dpre_w": 0x9000, "dpre_b": 0x901c}),
    ("two outputs", {"dgate": 0x9000, "dpost_w": 0x903c}), ("output is an input", {"dx": 0x4000 - 124}),
    ("output is an input", {"dh": "dn"}), ("output is an input", {"dgate": "post_w"}), ("output is an input", {"dpost_b": "gate"})])
def test_backward_refuses_overlaps(anywhere, why, change):
    names = ["r", "h", "gate", "gate_rows", "post_w", "post_b", "pre_w", "scale", "eps", "kind", "dr", "dn", "dx", "dh", "dgate",
             "dpost_w", "dpost_b", "dpre_w", "dpre_b", "rows", "cols", "accumulate"]
    args = {n: 0x100000 + 0x1000 * i for i, n in enumerate(names)}
    args.update(r=0x4000, gate_rows=2, scale=1.0, eps=1e-6, kind=1, rows=4, cols=8, accumulate=0)
    args.update({k: args[v] + 4 if isinstance(v, str) else v for k, v in change.items()})
    lib = cabi.load()
    assert lib.katsu_cuda_block_norm_bwd(anywhere, *(args[n] for n in names)) == cabi.ERR_INVALID_ARG
    assert why in lib.katsu_cuda_last_error_string().decode()
