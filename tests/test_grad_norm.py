"""The norm over many tensors, clipping and the clipped SGD step (katsu_cuda_grad_norm, _clip_grads, _sgd_step_clipped)."""
import ctypes

import numpy as np
import pytest

from katsu_b200 import cabi
from parity_util import DeviceArrays
from test_block_norm import anywhere  # noqa: F401 (fixture)

U = 2.0 ** -24

SIZES = {"one value": [1], "nothing": [], "empty ones": [0, 5, 0, 0, 3], "one chunk": [8192], "over a chunk": [8193, 8191, 1],
         "small CNN": [864, 18432, 65536 * 10], "many": [1 + (7 * i) % 23 for i in range(33)],
         "more than a launch takes": [3 + i % 5 for i in range(1100)], "launches in waves": [9001 + 4 * i for i in range(600)], "large": [3_000_001, 17, 2_500_000]}


def flat(sizes, seed, std=1.0):
    return (std * np.random.default_rng([seed, len(sizes)]).standard_normal(sum(sizes))).astype(np.float32)


def places(base, sizes, gap=0):
    """Addresses of tensors one right behind the other, `gap` floats apart."""
    return [base + 4 * (sum(sizes[:i]) + gap * i) for i in range(len(sizes))]


def factor(g, max_norm):
    norm = np.sqrt(np.square(g.astype(np.float64)).sum())
    return norm, np.float32(max_norm / norm) if norm > max_norm else np.float32(1)


@pytest.mark.gpu
@pytest.mark.parametrize("which", SIZES)
@pytest.mark.parametrize("share", [0.25, 3.0], ids=["clipped", "below"])
def test_norm_clip_and_step(ctx, which, share):
    sizes = SIZES[which]
    total = sum(sizes)
    g, w = flat(sizes, 1), flat(sizes, 2)
    norm, _ = factor(g, 1.0)
    max_norm = float(np.float32(share * norm))
    # The library divides 64-bit numbers and rounds once; its sum may differ in the last places of 64 bits, so its factor is
    # this one or a neighbour.
    c = factor(g, max_norm)[1]
    with DeviceArrays(ctx, g=np.append(g, 0), w=np.append(w, 0), n=np.zeros(1)) as d:
        d.alloc("out", total + 1, fill=9.0)
        gp, wp, op = (places(d[k], sizes) for k in ("g", "w", "out"))
        ctx.grad_norm(gp, sizes, d["n"])
        # a square root and one rounding behind a sum in 64 bits
        assert abs(d.get("n")[0] - norm) <= 2 * U * norm
        first = d.get("n")
        ctx.clip_grads(gp, op, sizes, max_norm, d["n"])
        assert np.array_equal(d.get("n"), first)
        out = d.get("out")
        assert out[total] == 9
        if c == 1:
            assert np.array_equal(out[:total], g)
        else:
            np.testing.assert_allclose(out[:total], g * np.float64(c), rtol=3 * U)  # factor, its neighbour, product
        ctx.sgd_step_clipped(wp, gp, sizes, 0.1, max_norm, d["n"])
        assert np.array_equal(d.get("n"), first)
        stepped = d.get("w")[:total]
        expect = w - np.float32(0.1) * out[:total]
        assert np.array_equal(stepped, expect)  # the bits of the two calls one after the other
        assert np.array_equal(d.get("g")[:total], g)
        ctx.clip_grads(gp, gp, sizes, max_norm, d["n"])
        assert np.array_equal(d.get("g")[:total], out[:total])


@pytest.mark.gpu
@pytest.mark.parametrize("gap_g,gap_w,shift", [(0, 0, 1), (1, 1, 0), (1, 2, 3), (3, 0, 2)])
def test_every_alignment(ctx, gap_g, gap_w, shift):
    """Gradients and weights at equal and at different places behind a 16-byte boundary; nothing around them changes."""
    sizes = [9001, 3, 40007, 2, 1, 16384]
    g, w = flat(sizes, 3), flat(sizes, 4)
    pad = 32

    def spread(v, gap, fill):
        a, at = np.full(v.size + gap * len(sizes) + pad, fill, np.float32), []
        for i, (n, p) in enumerate(zip(sizes, np.cumsum([0] + sizes[:-1]))):
            begin = shift + p + gap * i
            a[begin:begin + n] = v[p:p + n]
            at.append(begin)
        return a, at

    ga, gat = spread(g, gap_g, 1e30)
    wa, wat = spread(w, gap_w, 5.0)
    norm, c = factor(g, 20.0)
    with DeviceArrays(ctx, g=ga, w=wa, n=np.zeros(1)) as d:
        ctx.sgd_step_clipped([d["w"] + 4 * i for i in wat], [d["g"] + 4 * i for i in gat], sizes, 0.5, 20.0, d["n"])
        assert abs(d.get("n")[0] - norm) <= 2 * U * norm
        got, clipped = d.get("w"), g * c
        want = wa.copy()
        for n, p, b in zip(sizes, np.cumsum([0] + sizes[:-1]), wat):
            want[b:b + n] -= np.float32(0.5) * clipped[p:p + n]
        np.testing.assert_allclose(got, want, rtol=0, atol=4 * U * (np.abs(want).max() + np.abs(clipped).max()))
        outside = np.ones(wa.size, bool)
        for n, b in zip(sizes, wat):
            outside[b:b + n] = False
        assert (got[outside] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-44, 1e25])
def test_squares_beyond_f32(ctx, scale):
    g = (np.arange(1, 5001) * np.float64(scale)).astype(np.float32)
    norm = np.sqrt(np.square(g.astype(np.float64)).sum())
    with DeviceArrays(ctx, g=g, n=np.zeros(1)) as d:
        ctx.grad_norm([d["g"]], [g.size], d["n"])
        got = d.get("n")[0]
    assert abs(got - norm) <= 2 * U * norm + 2.0 ** -150


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_not_finite(ctx, bad):
    sizes = [5000, 9000]
    g, w = flat(sizes, 5), flat(sizes, 6)
    g[7001] = bad
    with DeviceArrays(ctx, g=g, w=w, n=np.zeros(1)) as d:
        d.alloc("out", g.size, fill=0.0)
        gp = places(d["g"], sizes)
        ctx.clip_grads(gp, places(d["out"], sizes), sizes, 1.0, d["n"])
        assert not np.isfinite(d.get("n")[0])
        assert np.array_equal(d.get("out"), g, equal_nan=True)
        ctx.clip_grads(gp, gp, sizes, 1.0, d["n"])
        assert np.array_equal(d.get("g"), g, equal_nan=True)
        ctx.sgd_step_clipped(places(d["w"], sizes), gp, sizes, 0.1, 1.0, d["n"])
        assert np.array_equal(d.get("w"), w)


@pytest.mark.gpu
def test_norm_at_the_limit_changes_nothing(ctx):
    g = np.array([3.0, 4.0], np.float32)
    with DeviceArrays(ctx, g=g, n=np.zeros(1)) as d:
        ctx.clip_grads([d["g"]], [d["g"]], [2], 5.0, d["n"])
        assert d.get("n")[0] == 5 and np.array_equal(d.get("g"), g)
        ctx.clip_grads([d["g"]], [d["g"]], [2], float(np.nextafter(np.float32(5), np.float32(0))), d["n"])
        assert not np.array_equal(d.get("g"), g)


@pytest.mark.gpu
def test_limits_of_zero_and_infinity(ctx):
    g = flat([1000], 7)
    with DeviceArrays(ctx, g=g, n=np.zeros(1)) as d:
        ctx.clip_grads([d["g"]], [d["g"]], [1000], float("inf"), d["n"])
        assert np.array_equal(d.get("g"), g)
        ctx.clip_grads([d["g"]], [d["g"]], [1000], 0.0, d["n"])
        assert not d.get("g").any()
        ctx.clip_grads([d["g"]], [d["g"]], [1000], 0.0, d["n"])  # a norm of 0 is not above 0
        assert d.get("n")[0] == 0 and not d.get("g").any()


@pytest.mark.gpu
def test_replayed_and_on_other_streams():
    from test_captured_calls import capture

    sizes = SIZES["small CNN"]
    g, w = flat(sizes, 8), flat(sizes, 9)
    contexts, results = [cabi.Context(0) for _ in range(2)], []
    try:
        for c in contexts:
            with DeviceArrays(c, g=g, w=w, n=np.zeros(1)) as d:
                def call():
                    c.sgd_step_clipped(places(d["w"], sizes), places(d["g"], sizes), sizes, 0.1, 3.0, d["n"])

                call()
                eager = d.get("w"), d.get("n")
                replay = capture(c, call)
                for scale in (2.0, 1.0):  # a replay looks at its own gradients
                    c.h2d(d["w"], w), c.h2d(d["g"], g * np.float32(scale))
                    c.sync()
                    replay()
                    got = d.get("w"), d.get("n")
                    assert got[1][0] == np.float32(scale) * eager[1][0]
                assert np.array_equal(got[0], eager[0])
                del replay
                results.append(eager[0])
        assert np.array_equal(*results)
    finally:
        for c in contexts:
            c.close()


def arrays(pointers, counts):
    return (ctypes.c_void_p * max(1, len(pointers)))(*pointers), (ctypes.c_size_t * max(1, len(counts)))(*counts)


@pytest.mark.parametrize("why,weights,grads,counts,max_norm,norm", [
    ("norm is null", [0x10000], [0x20000], [4], 1.0, None),
    ("max_norm", [0x10000], [0x20000], [4], -1.0, 0x90000),
    ("max_norm", [0x10000], [0x20000], [4], float("nan"), 0x90000),
    ("null gradient", [0x10000], [None], [4], 1.0, 0x90000),
    ("null output or weight", [None], [0x20000], [4], 1.0, 0x90000),
    ("whole float", [0x10002], [0x20000], [4], 1.0, 0x90000),
    ("whole float", [0x10000], [0x20001], [4], 1.0, 0x90000),
    ("count", [0x10000], [0x20000], [1 << 62], 1.0, 0x90000),
    ("overlap", [0x10000, 0x10000], [0x20000, 0x30000], [4, 4], 1.0, 0x90000),
    ("overlap", [0x10000, 0x1000c], [0x20000, 0x30000], [4, 4], 1.0, 0x90000),
    ("overlap", [0x10000, 0x20000], [0x20000, 0x30000], [4, 4], 1.0, 0x90000),
    ("overlap", [0x10000], [0x10000], [4], 1.0, 0x90000),
    ("overlap", [0x10000], [0x0fff4], [4], 1.0, 0x90000),
    ("norm lies", [0x10000], [0x20000], [4], 1.0, 0x20008),
    ("norm lies", [0x10000], [0x20000], [4], 1.0, 0x1000c),
])
def test_step_refuses(anywhere, why, weights, grads, counts, max_norm, norm):  # noqa: F811
    lib = cabi.load()
    w, c = arrays(weights, counts)
    g, _ = arrays(grads, counts)
    assert lib.katsu_cuda_sgd_step_clipped(anywhere, w, g, c, len(counts), 0.1, max_norm, norm) == cabi.ERR_INVALID_ARG
    assert why in lib.katsu_cuda_last_error_string().decode()


@pytest.mark.parametrize("why,out,grads", [
    ("overlap", [0x20000, 0x30000], [0x30000, 0x20000]),  # another's place
    ("overlap", [0x20004, 0x30000], [0x20000, 0x30000]),  # its own, moved
    ("overlap", [0x20000, 0x20000], [0x20000, 0x20000]),  # the same gradient twice
])
def test_clip_refuses(anywhere, why, out, grads):  # noqa: F811
    lib = cabi.load()
    o, c = arrays(out, [4, 4])
    g, _ = arrays(grads, [4, 4])
    assert lib.katsu_cuda_clip_grads(anywhere, g, o, c, 2, 1.0, 0x90000) == cabi.ERR_INVALID_ARG
    assert why in lib.katsu_cuda_last_error_string().decode()
    assert lib.katsu_cuda_clip_grads(None, g, o, c, 2, 1.0, 0x90000) == cabi.ERR_INVALID_ARG


def test_lists_of_different_lengths_are_refused():
    class Nothing(cabi.Context):
        def __init__(self):
            pass

        def call(self, *args):
            raise AssertionError("reached the library")

    for call in (lambda c: c.grad_norm([1, 2], [3], 4), lambda c: c.clip_grads([1], [1, 2], [3], 1.0, 4),
                 lambda c: c.sgd_step_clipped([1, 2], [1], [3], 0.1, 1.0, 4), lambda c: c.clip_grads([1], [1], [3, 3], 1.0, 4)):
        with pytest.raises(ValueError):
            call(Nothing())


@pytest.mark.parametrize("norm", [0x90001, 0x90002, 0x90003])
def test_a_norm_between_two_floats_is_refused(anywhere, norm):  # noqa: F811
    lib = cabi.load()
    (w, c), (g, _) = arrays([0x10000], [4]), arrays([0x20000], [4])
    for call in (lambda: lib.katsu_cuda_grad_norm(anywhere, g, c, 1, norm), lambda: lib.katsu_cuda_clip_grads(anywhere, g, w, c, 1, 1.0, norm),
                 lambda: lib.katsu_cuda_sgd_step_clipped(anywhere, w, g, c, 1, 0.1, 1.0, norm)):
        assert call() == cabi.ERR_INVALID_ARG
        assert "whole float" in lib.katsu_cuda_last_error_string().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1001], [5000, 9001, 3]], ids=str)
@pytest.mark.parametrize("shift", [0, 1])
def test_values_that_stay_keep_their_bits(ctx, sizes, shift):
    """Below the limit and beside a gradient that is no number: signs of zeros, NaNs' bits and the smallest numbers arrive as they are."""
    bits = np.random.default_rng(11).integers(0, 2 ** 32, sum(sizes), dtype=np.uint32)
    small = np.where(np.arange(bits.size) % 3 == 0, bits & np.uint32(0x80000000), bits & np.uint32(0x807fffff))
    for v in (bits, small):  # any values, NaNs among them; zeros and subnormal numbers
        with DeviceArrays(ctx, g=v.view(np.float32), n=np.zeros(1)) as d:
            d.alloc("out", bits.size + 4, fill=0.0)
            ctx.clip_grads(places(d["g"], sizes), places(d["out"] + 4 * shift, sizes), sizes, 1.0, d["n"])
            assert np.array_equal(d.get("out")[shift:shift + bits.size].view(np.uint32), v)
            assert np.isnan(d.get("n")[0]) == (v is bits)
