"""The product in 8-bit integers (katsu_cuda_int8_*): whole numbers equal to the definition's, results to their roundings."""
import ctypes

import numpy as np
import pytest

import block_ref
from katsu_b200 import cabi
from parity_util import DeviceArrays
from test_block_norm import anywhere  # noqa: F401 (fixture)

U = 2.0 ** -24


def pitch(k):
    return (k + 15) // 16 * 16


def floats(rows, k):
    return rows * pitch(k) // 4


def values(rows, k, seed=0):
    rng = np.random.default_rng([seed, rows, k])
    v = rng.standard_normal((rows, k)) * np.where(rng.random(k) < 0.02, 10.0, 1.0)
    return v.astype(np.float32)


def whole(d, name, rows, k):
    """A quantised matrix, its padding held to zero."""
    q = d.get(name)[:floats(rows, k)].view(np.int8).reshape(rows, pitch(k))
    assert not q[:, k:].any()
    return q[:, :k].astype(np.int64)


def check_result(y, xq, xs, wq, ws, bias):
    """Four roundings: the sum's conversion, two products, and the sum with the bias."""
    want = block_ref.int8_product(xq, xs, wq, ws, None)
    b = 0.0 if bias is None else bias.astype(np.float64)
    bound = 3.01 * U * np.abs(want) + U * (np.abs(want + b) + 3.01 * U * np.abs(want)) + 2.0 ** -149
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(y), bad)
    off = np.abs(y.astype(np.float64) - (want + b))
    assert (off <= bound)[~bad].all(), (np.argwhere(~(off <= bound) & ~bad)[:5], (off - bound)[~bad].max())


SHAPES = [(1, 1, 1), (1, 16, 1), (1, 4096, 4096), (2, 100, 33), (3, 17, 5), (4, 513, 129), (5, 2048, 70), (7, 31, 300),
          (8, 1024, 515), (1, 20000, 3), (2, 60001, 10), (8, 4096, 1000), (9, 64, 40), (16, 128, 256), (16, 144, 257),
          (33, 500, 100), (64, 4096, 128), (100, 1031, 517), (130, 257, 255), (256, 384, 512), (300, 2047, 515),
          (512, 8192, 10), (1021, 333, 700), (40, 30000, 24), (1, 133144, 2), (12, 133144, 3), (5, 16384, 2056), (160, 20000, 8),
          (300, 9000, 8), (1300, 1100, 8), (4000, 100, 16), (700, 5000, 12), (100, 20001, 8), (20, 65536, 10), (60, 60001, 8),
          (25, 70001, 5), (320, 40000, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product(ctx, m, k, n):
    x, w = values(m, k, 1), values(k, n, 2)
    bias = None if (m + n) % 2 else values(1, n, 3)[0]
    xq, xs = block_ref.quantize(x)
    wq, ws = block_ref.quantize(w.T)
    with DeviceArrays(ctx, x=x, w=w, **({} if bias is None else {"bias": bias})) as d:
        for name, count in (("wq", floats(n, k)), ("ws", n), ("xq", floats(m, k)), ("xs", m), ("y", m * n + 8), ("y2", m * n)):
            d.alloc(name, count, fill=np.nan)
        b = None if bias is None else d["bias"]
        ctx.int8_quantize_weights(d["w"], d["wq"], d["ws"], k, n)
        assert np.array_equal(whole(d, "wq", n, k), wq) and np.array_equal(d.get("ws"), ws)
        ctx.int8_quantize_rows(d["x"], d["xq"], d["xs"], m, k)
        assert np.array_equal(whole(d, "xq", m, k), xq) and np.array_equal(d.get("xs"), xs)
        ctx.int8_linear(d["x"], d["wq"], d["ws"], b, d["y"], m, k, n)
        y = d.get("y")
        assert np.isnan(y[m * n:]).all()  # what lies behind the result
        check_result(y[:m * n].reshape(m, n), xq, xs, wq, ws, bias)
        ctx.int8_matmul(d["xq"], d["xs"], d["wq"], d["ws"], b, d["y2"], m, k, n)
        assert np.array_equal(d.get("y2"), y[:m * n])


def test_row_bytes():
    lib, out = cabi.load(), ctypes.c_size_t(0)
    for k in (1, 15, 16, 17, cabi.INT8_MAX_K):
        assert lib.katsu_cuda_int8_row_bytes(k, ctypes.byref(out)) == cabi.OK and out.value == pitch(k)
    for k in (0, cabi.INT8_MAX_K + 1):
        assert lib.katsu_cuda_int8_row_bytes(k, ctypes.byref(out)) == cabi.ERR_INVALID_ARG
    assert lib.katsu_cuda_int8_row_bytes(1, None) == cabi.ERR_INVALID_ARG


def borders(k, seed):
    """Rows whose quotients lie on borders between whole numbers and one place to either side of them."""
    rng = np.random.default_rng(seed)
    rows = []
    for exponent in (0, -20, 40, -125, -140, 120):
        top = np.float32(np.ldexp(127.0 if exponent == 0 else 100 + 27 * rng.random(), exponent))
        scale = top / np.float32(127)
        n = rng.integers(-127, 127, k) + 0.5
        v = (n * np.float64(scale)).astype(np.float32)
        v = np.where(rng.random(k) < 0.3, np.nextafter(v, np.float32(0)), np.where(rng.random(k) < 0.3, np.nextafter(v, np.float32(np.inf)), v))
        v = np.clip(v, -top, top)
        v[rng.integers(0, k)] = top
        rows.append(v.astype(np.float32))
    return np.stack(rows)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [64, 1000, 1025, 9001])
def test_borders_ties_and_ranges(ctx, k):
    x = borders(k, k)
    x[4, : k // 2] = np.float32(1e-45)  # places of the smallest numbers
    xq, xs = block_ref.quantize(x)
    m = len(x)
    with DeviceArrays(ctx, x=x, w=np.ascontiguousarray(x.T)) as d:
        for name, count in (("xq", floats(m, k)), ("xs", m), ("wq", floats(m, k)), ("ws", m)):
            d.alloc(name, count, fill=np.nan)
        ctx.int8_quantize_rows(d["x"], d["xq"], d["xs"], m, k)
        assert np.array_equal(d.get("xs"), xs) and np.array_equal(whole(d, "xq", m, k), xq)
        ctx.int8_quantize_weights(d["w"], d["wq"], d["ws"], k, m)
        assert np.array_equal(d.get("ws"), xs) and np.array_equal(whole(d, "wq", m, k), xq)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 6, 40])
def test_rows_that_have_no_scale(ctx, m):
    """Zeros, infinities, NaNs and the smallest numbers, in a token and in a channel, stay with it."""
    k, n = 300, 37
    x, w = values(m, k, 4), values(k, n, 5)
    x[0, 5] = np.nan
    if m > 1:
        x[1], x[2, 7], x[3] = 0.0, -np.inf, np.float32(1e-45)
    w[:, 2], w[9, 3], w[0, 4] = 0.0, np.inf, np.nan
    xq, xs = block_ref.quantize(x)
    wq, ws = block_ref.quantize(w.T)
    with DeviceArrays(ctx, x=x, w=w) as d:
        for name, count in (("wq", floats(n, k)), ("ws", n), ("y", m * n)):
            d.alloc(name, count, fill=0.0)
        ctx.int8_quantize_weights(d["w"], d["wq"], d["ws"], k, n)
        assert np.array_equal(d.get("ws"), ws, equal_nan=True)
        ctx.int8_linear(d["x"], d["wq"], d["ws"], None, d["y"], m, k, n)
        check_result(d.get("y").reshape(m, n), xq, xs, wq, ws, None)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(3, 130, 50), (60, 130, 50), (200, 1000, 300)])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_unaligned(ctx, m, k, n, shift):
    """x, scales, bias and y at any float; results of a token alone and among others have the same bits."""
    x, w, bias = values(m, k, 6), values(k, n, 7), values(1, n, 8)[0]
    xq, xs = block_ref.quantize(x)
    wq, ws = block_ref.quantize(w.T)
    pad = lambda v: np.concatenate([np.zeros(shift, np.float32), v.reshape(-1)])  # noqa: E731
    s = 4 * shift
    with DeviceArrays(ctx, x=pad(x), w=pad(w), bias=pad(bias)) as d:
        for name, count in (("wq", floats(n, k)), ("ws", n + shift), ("y", m * n + 8), ("one", n)):
            d.alloc(name, count, fill=3.0)
        ctx.int8_quantize_weights(d["w"] + s, d["wq"], d["ws"] + s, k, n)
        ctx.int8_linear(d["x"] + s, d["wq"], d["ws"] + s, d["bias"] + s, d["y"] + s, m, k, n)
        got = d.get("y")
        assert (got[:shift] == 3).all() and (got[shift + m * n:] == 3).all()
        y = got[shift:shift + m * n].reshape(m, n)
        check_result(y, xq, xs, wq, ws, bias)
        for i in (0, m - 1):
            ctx.int8_linear(d["x"] + s + 4 * k * i, d["wq"], d["ws"] + s, d["bias"] + s, d["one"], 1, k, n)
            assert np.array_equal(d.get("one"), y[i])


@pytest.mark.gpu
def test_largest_sums(ctx):
    """All magnitudes at 127, the longest k: the sum ends just below 2^31."""
    k = cabi.INT8_MAX_K
    for m, n in ((1, 2), (20, 3)):
        x, w = np.ones((m, k), np.float32), np.ones((k, n), np.float32)
        w[:, 1] = -1.0
        with DeviceArrays(ctx, x=x, w=w) as d:
            for name, count in (("wq", floats(n, k)), ("ws", n), ("y", m * n)):
                d.alloc(name, count, fill=0.0)
            ctx.int8_quantize_weights(d["w"], d["wq"], d["ws"], k, n)
            ctx.int8_linear(d["x"], d["wq"], d["ws"], None, d["y"], m, k, n)
            y = d.get("y").reshape(m, n)
        want = np.full((m, n), float(k))
        want[:, 1] = -k
        np.testing.assert_allclose(y, want, rtol=6 * U)  # two scales of 1 / 127, conversion, two products


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(0, 4), (4, 0)])
def test_nothing_to_do(ctx, m, n):
    with DeviceArrays(ctx, a=np.ones(64)) as d:
        d.alloc("y", 16, fill=2.0)
        ctx.int8_linear(d["a"], d["a"], d["a"], None, d["y"], m, 16, n)
        ctx.int8_matmul(d["a"], d["a"], d["a"], d["a"], None, d["y"], m, 16, n)
        ctx.int8_quantize_rows(d["a"], d["y"], d["y"], 0, 16)
        ctx.int8_quantize_weights(d["a"], d["y"], d["y"], 16, 0)
        assert (d.get("y") == 2).all()


# With 148 SMs: tiles of 32 to 256 tokens, each in two or more rounds (accumulators and the ring's stages go from tile to tile, the last
# round is not full), and tiles of 128 to 256 with k split.
@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(1600, 230, 544), (3372, 247, 584), (3501, 278, 515), (4027, 262, 1319), (2500, 1300, 2100), (4063, 268, 1627),
                                   (2000, 700, 3000), (4195, 266, 2105), (4271, 270, 2798), (3905, 290, 4441), (1161, 5792, 282), (774, 12396, 274),
                                   (536, 18790, 522), (1296, 17479, 269), (1748, 17120, 258)])
def test_many_tokens(ctx, m, k, n):
    x, w, bias = values(m, k, 13), values(k, n, 14), values(1, n, 15)[0]
    xq, xs = block_ref.quantize(x)
    wq, ws = block_ref.quantize(w.T)
    with DeviceArrays(ctx, x=x, w=w, bias=bias) as d:
        for name, count in (("wq", floats(n, k)), ("ws", n), ("y", m * n + 8)):
            d.alloc(name, count, fill=np.nan)
        ctx.int8_quantize_weights(d["w"], d["wq"], d["ws"], k, n)
        ctx.int8_linear(d["x"], d["wq"], d["ws"], d["bias"], d["y"], m, k, n)
        y = d.get("y")
    assert np.isnan(y[m * n:]).all()
    check_result(y[:m * n].reshape(m, n), xq.astype(np.float64), xs, wq.astype(np.float64), ws, bias)  # (sums below 2^53 are exact)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(1, 4096, 512), (8, 8192, 300), (300, 1024, 600), (32, 8192, 256)])
def test_replayed_and_on_other_streams(m, k, n):
    from test_captured_calls import capture

    x, w = values(m, k, 9), values(k, n, 10)
    contexts, results = [cabi.Context(0) for _ in range(2)], []
    try:
        for c in contexts:
            with DeviceArrays(c, x=x, w=w) as d:
                for name, count in (("wq", floats(n, k)), ("ws", n), ("y", m * n)):
                    d.alloc(name, count, fill=0.0)
                c.int8_quantize_weights(d["w"], d["wq"], d["ws"], k, n)
                call = lambda: c.int8_linear(d["x"], d["wq"], d["ws"], None, d["y"], m, k, n)  # noqa: E731
                call()
                eager = d.get("y")
                replay = capture(c, call)
                c.h2d(d["x"], x * np.float32(4))
                c.sync()
                replay()
                assert np.array_equal(d.get("y"), 4 * eager)  # scales are of the replay's own x
                del replay
                results.append(eager)
        assert np.array_equal(*results)
    finally:
        for c in contexts:
            c.close()


A = [0x10000 * (i + 1) for i in range(6)]


@pytest.mark.parametrize("name,why,args", [
    ("linear", "k must", (A[0], A[1], A[2], None, A[3], 4, 0, 4)),
    ("linear", "k must", (A[0], A[1], A[2], None, A[3], 4, cabi.INT8_MAX_K + 1, 4)),
    ("linear", "too many", (A[0], A[1], A[2], None, A[3], 1 << 30, 4, 4)),
    ("linear", "too many", (A[0], A[1], A[2], None, A[3], 4, 4, 1 << 30)),
    ("linear", "null", (None, A[1], A[2], None, A[3], 4, 4, 4)),
    ("linear", "null", (A[0], None, A[2], None, A[3], 4, 4, 4)),
    ("linear", "null", (A[0], A[1], None, None, A[3], 4, 4, 4)),
    ("linear", "null", (A[0], A[1], A[2], None, None, 4, 4, 4)),
    ("linear", "aligned", (A[0], A[1] + 8, A[2], None, A[3], 4, 4, 4)),
    ("linear", "input", (A[0], A[1], A[2], None, A[0], 4, 4, 4)),
    ("matmul", "null", (A[0], None, A[1], A[2], None, A[3], 4, 4, 4)),
    ("matmul", "aligned", (A[0] + 4, A[4], A[1], A[2], None, A[3], 4, 4, 4)),
    ("matmul", "input", (A[0], A[4], A[1], A[2], A[3], A[3], 4, 4, 4)),
    ("quantize_rows", "k must", (A[0], A[1], A[2], 4, 0)),
    ("quantize_rows", "null", (A[0], A[1], None, 4, 4)),
    ("quantize_rows", "aligned", (A[0], A[1] + 1, A[2], 4, 4)),
    ("quantize_rows", "too many", (A[0], A[1], A[2], 1 << 31, 4)),
    ("quantize_weights", "k must", (A[0], A[1], A[2], cabi.INT8_MAX_K + 1, 4)),
    ("quantize_weights", "null", (A[0], None, A[2], 4, 4)),
    ("quantize_weights", "aligned", (A[0], A[1] + 12, A[2], 4, 4)),
    ("quantize_weights", "too many", (A[0], A[1], A[2], 4, 1 << 31)),
])
def test_refusals(anywhere, name, why, args):  # noqa: F811
    lib = cabi.load()
    call = getattr(lib, "katsu_cuda_int8_" + name)
    assert call(anywhere, *args) == cabi.ERR_INVALID_ARG
    assert why in lib.katsu_cuda_last_error_string().decode()
    assert call(None, *args) == cabi.ERR_INVALID_ARG


# m = 8, k = 20, n = 6: x 640 bytes, y 192, a quantised row 32
@pytest.mark.parametrize("name,args", [
    ("linear", (A[0], A[1], A[2], None, A[0] + 636, 8, 20, 6)), ("linear", (A[0], A[1], A[2], None, A[0] - 188, 8, 20, 6)),
    ("linear", (A[0], A[1], A[2], None, A[1] + 188, 8, 20, 6)), ("linear", (A[0], A[1], A[2], None, A[2] + 20, 8, 20, 6)),
    ("linear", (A[0], A[1], A[2], A[3], A[3] - 188, 8, 20, 6)), ("matmul", (A[0], A[4], A[1], A[2], A[3], A[0] + 252, 8, 20, 6)),
    ("matmul", (A[0], A[4], A[1], A[2], A[3], A[4] + 28, 8, 20, 6)), ("quantize_rows", (A[0], A[0], A[1], 8, 20)),
    ("quantize_rows", (A[0], A[0] + 624, A[1], 8, 20)), ("quantize_rows", (A[0], A[0] - 240, A[1], 8, 20)),
    ("quantize_rows", (A[0], A[1], A[0] + 636, 8, 20)), ("quantize_rows", (A[0], A[1], A[1] + 252, 8, 20)),
    ("quantize_weights", (A[0], A[0] + 464, A[1], 20, 6)), ("quantize_weights", (A[0], A[1], A[0] - 20, 20, 6)),
    ("quantize_weights", (A[0], A[1], A[1] - 20, 20, 6)),
])
def test_overlaps_are_refused(anywhere, name, args):  # noqa: F811
    lib = cabi.load()
    assert getattr(lib, "katsu_cuda_int8_" + name)(anywhere, *args) == cabi.ERR_INVALID_ARG
    assert "input" in lib.katsu_cuda_last_error_string().decode()


# Rows of the few-token kernel in shared memory: a launch's dynamic part on both sides of 48 KiB less the kernel's static part, and of
# 48 KiB itself.  A process of its own for each: the first launch of a kernel must not depend on a larger one before it.
@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(1, 49024, 8), (1, 49152, 8), (1, 49153, 8), (2, 24464, 16), (2, 24576, 16), (2, 24577, 16), (3, 12177, 9),
                                   (4, 12288, 64), (4, 12289, 64), (5, 6033, 33), (8, 6144, 64), (8, 6145, 64)])
def test_first_call_of_a_process(m, k, n):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, __file__, str(m), str(k), str(n)], capture_output=True, text=True, timeout=300,
                         env=dict(os.environ, PYTHONPATH=root))
    assert run.returncode == 0, run.stderr[-2000:]


def first_call(m, k, n):
    x, w = values(m, k, 11), values(k, n, 12)
    xq, xs = block_ref.quantize(x)
    wq, ws = block_ref.quantize(w.T)
    laid = np.zeros((n, pitch(k)), np.int8)
    laid[:, :k] = wq
    rows = np.zeros((m, pitch(k)), np.int8)
    rows[:, :k] = xq
    ctx = cabi.Context(0)
    with DeviceArrays(ctx, x=x, wq=laid.view(np.float32), ws=ws, xq=rows.view(np.float32), xs=xs) as d:
        d.alloc("y", m * n, fill=np.nan)
        ctx.int8_matmul(d["xq"], d["xs"], d["wq"], d["ws"], None, d["y"], m, k, n)
        check_result(d.get("y").reshape(m, n), xq, xs, wq, ws, None)
        d.alloc("y2", m * n, fill=np.nan)
        ctx.int8_linear(d["x"], d["wq"], d["ws"], None, d["y2"], m, k, n)
        assert np.array_equal(d.get("y2"), d.get("y"))
    ctx.close()


if __name__ == "__main__":
    import sys

    first_call(*(int(v) for v in sys.argv[1:]))
