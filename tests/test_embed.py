"""Rows of a table for tokens, from f32 and from 8 bits, and the gradient of the table (katsu_cuda_embed_*, _int8_embed)."""
import numpy as np
import pytest

import vocab_ref as ref
from katsu_b200 import cabi
from parity_util import DeviceArrays
from test_block_norm import anywhere  # noqa: F401 (fixture)
from test_int8 import floats, pitch

NONE = [-1, -2 ** 31, 2 ** 31 - 1]  # no tokens, whatever the vocabulary


def some_tokens(rng, count, vocab, how="zipf"):
    if how == "one":
        return np.full(count, vocab - 1)
    tokens = ref.zipf(rng, vocab, count) if how == "zipf" else rng.integers(0, vocab, count)
    if how == "holes":
        tokens[rng.random(count) < 0.3] = -1
        tokens[: min(count, 4)] = [vocab, *NONE][: min(count, 4)]
    if how == "half":  # a padding token
        tokens[rng.random(count) < 0.7] = min(1, vocab - 1)
    if how == "blocks":  # runs that end with whole pieces and bundles of them
        tokens = np.arange(count) * vocab // count
        rng.shuffle(tokens)
    if how == "sorted":
        tokens.sort()
    return tokens


LOOKUPS = [(1, 1, 1), (1, 5, 4096), (3, 7, 3), (17, 100, 16), (33, 50, 515), (2, 9, 8200), (1000, 300, 64), (129, 64, 1028), (70, 33, 5000),
           (257, 1000, 20), (4, 3, 40001)]


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [(0, 0), (1, 0), (0, 3), (2, 2)], ids=str)
@pytest.mark.parametrize("count,vocab,cols", LOOKUPS)
def test_lookup(ctx, count, vocab, cols, shift):
    rng = np.random.default_rng([count, vocab, cols])
    table = rng.standard_normal((vocab, cols)).astype(np.float32)
    tokens = some_tokens(rng, count, vocab, "holes")
    scale = np.float32(cols ** 0.5)
    with DeviceArrays(ctx, table=np.concatenate([np.zeros(shift[0], np.float32), table.reshape(-1)]), tokens=ref.device_ints(tokens)) as d:
        d.alloc("y", count * cols + 8, fill=np.nan)
        ctx.embed_fwd(d["table"] + 4 * shift[0], d["tokens"], scale, d["y"] + 4 * shift[1], count, vocab, cols)
        y = d.get("y")
    assert np.isnan(y[: shift[1]]).all() and np.isnan(y[shift[1] + count * cols:]).all()
    # one rounding
    assert np.array_equal(y[shift[1]: shift[1] + count * cols].reshape(count, cols), ref.embed(table, tokens, float(scale)).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1, 2])
@pytest.mark.parametrize("count,vocab,cols", LOOKUPS)
def test_lookup_in_8_bits(ctx, count, vocab, cols, shift):
    """From the weights of a head [cols, vocab], quantised as the 8-bit product keeps them."""
    rng = np.random.default_rng([count, vocab, cols, 1])
    w = rng.standard_normal((cols, vocab)).astype(np.float32)
    tokens = some_tokens(rng, count, vocab, "holes")
    scale = np.float32(1.7)
    with DeviceArrays(ctx, w=w, tokens=ref.device_ints(tokens)) as d:
        d.alloc("q", floats(vocab, cols)), d.alloc("s", vocab), d.alloc("y", count * cols + 8, fill=np.nan)
        ctx.int8_quantize_weights(d["w"], d["q"], d["s"], cols, vocab)
        ctx.int8_embed(d["q"], d["s"], d["tokens"], scale, d["y"] + 4 * shift, count, vocab, cols)
        q = d.get("q")[: floats(vocab, cols)].view(np.int8).reshape(vocab, pitch(cols))[:, :cols]
        s, y = d.get("s"), d.get("y")
    there = ref.valid(tokens, vocab)
    at = np.where(there, tokens, 0)
    want = np.where(there[:, None], (q[at].astype(np.float32) * s[at][:, None]) * scale, np.float32(0))
    assert np.isnan(y[:shift]).all() and np.isnan(y[shift + count * cols:]).all()
    assert np.array_equal(y[shift: shift + count * cols].reshape(count, cols), want)


@pytest.mark.gpu
def test_lookup_of_no_tokens_and_in_no_table(ctx):
    with DeviceArrays(ctx, t=ref.device_ints([0, -1, 5])) as d:
        d.alloc("y", 12, fill=np.nan)
        ctx.embed_fwd(None, d["t"], 2.0, d["y"], 0, 0, 4)
        ctx.embed_fwd(None, d["t"], 2.0, d["y"], 3, 9, 0)
        assert np.isnan(d.get("y")).all()
        ctx.embed_fwd(None, d["t"], 2.0, d["y"], 3, 0, 4)
        assert not d.get("y").any()


# counts up to and above 256, to which tokens are not sorted, around 8192, where the sort changes, and 4096 and more, where pieces grow; runs of more than 32 pieces; vocabularies of
# one to three digits of a sort
GRADS = [(127, 9, 24, "zipf"), (128, 3, 40, "one"), (128, 500, 513, "holes"), (129, 3, 40, "one"), (256, 2, 516, "uniform"), (256, 90, 64, "zipf"), (257, 2, 516, "uniform"), (255, 1, 3, "one"), (160, 1, 12, "one"), (161, 300, 515, "holes"),
         (40000, 5, 8, "half"), (40000, 2, 1030, "half"), (66000, 3, 36, "half"), (16384 + 512, 2, 8, "blocks"), (65536, 4, 12, "blocks"),
         (4096, 30, 20, "zipf"), (16384, 2, 12, "uniform"), (16385, 9, 12, "zipf"), (65537, 5, 4, "zipf"), (32768, 3, 8, "one"), (32769, 3, 8, "one"), (32800, 100, 132, "zipf"), (50000, 2, 1, "uniform"),
         (1, 1, 1, "one"), (2, 3, 5, "zipf"), (31, 1, 4, "one"), (32, 2, 4, "uniform"), (33, 1, 7, "one"), (64, 9, 16, "sorted"),
         (65, 200, 36, "holes"), (100, 40, 515, "zipf"), (1000, 10, 64, "zipf"), (1000, 5000, 1030, "uniform"), (300, 7, 4100, "zipf"),
         (4097, 100, 20, "one"), (8191, 1000, 8, "zipf"), (8192, 50, 12, "holes"), (8193, 1023, 12, "zipf"), (8193, 1024, 5, "holes"),
         (9000, 1, 33, "one"), (20000, 70000, 4, "zipf"), (30001, 3000, 40, "sorted"), (70000, 500, 3, "uniform"), (12345, 1 << 20, 4, "zipf"),
         (9999, (1 << 20) + 5, 3, "holes"), (300000, 40000, 4, "zipf"), (40, 2000, 2, "holes")]


def check_grad(ctx, count, vocab, cols, how, shift, accumulate):
    rng = np.random.default_rng([count, vocab, cols])
    tokens, dy = some_tokens(rng, count, vocab, how), rng.standard_normal((count, cols)).astype(np.float32)
    before = rng.standard_normal((vocab, cols)).astype(np.float32)
    scale = np.float32(0.37)
    want, off = ref.embed_grad(tokens, dy, float(scale), vocab)
    start = before if accumulate else np.full((vocab, cols), np.nan, np.float32)
    edge = np.full(4, 7.0, np.float32)
    with DeviceArrays(ctx, tokens=ref.device_ints(tokens), dy=np.concatenate([edge[:shift], dy.reshape(-1)]),
                      table=np.concatenate([edge[:shift], start.reshape(-1), edge])) as d:
        ctx.embed_bwd(d["tokens"], d["dy"] + 4 * shift, scale, d["table"] + 4 * shift, count, vocab, cols, accumulate)
        got = d.get("table")
    assert (got[:shift] == 7).all() and (got[shift + vocab * cols:] == 7).all()
    got = got[shift: shift + vocab * cols].reshape(vocab, cols)
    untouched = np.ones(vocab, bool)
    untouched[tokens[ref.valid(tokens, vocab)]] = False
    if accumulate:
        assert np.array_equal(got[untouched], before[untouched])
        want, off = want + before, off + 1.01 * ref.U * np.abs(want + before)
    else:
        assert not got[untouched].any()
    ref.assert_near(got[~untouched], want[~untouched], off[~untouched])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("count,vocab,cols,how", GRADS)
def test_gradient(ctx, count, vocab, cols, how, accumulate):
    check_grad(ctx, count, vocab, cols, how, 0, accumulate)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("count,vocab,cols", [(200, 30, 64), (9000, 300, 16), (77, 5, 1024)])
def test_gradient_at_any_address(ctx, count, vocab, cols, shift):
    for accumulate in (0, 1):
        # the order of the sums does not depend on addresses
        assert np.array_equal(check_grad(ctx, count, vocab, cols, "zipf", shift, accumulate),
                              check_grad(ctx, count, vocab, cols, "zipf", 0, accumulate))


@pytest.mark.gpu
@pytest.mark.parametrize("count,cols", [(50000, 512), (40000, 260), (20000, 16), (100000, 20)])
def test_gradient_of_many_tokens_at_any_address(ctx, count, cols):
    """The same bits, where rows that are whole 16-byte units have other threads than those that are not."""
    assert np.array_equal(check_grad(ctx, count, 300, cols, "zipf", 1, 0), check_grad(ctx, count, 300, cols, "zipf", 0, 0))


@pytest.mark.gpu
def test_gradient_of_no_tokens(ctx):
    with DeviceArrays(ctx, t=ref.device_ints([-1] * 40), dy=np.ones(160)) as d:
        for count in (0, 40):
            d.alloc("g", 20, fill=np.nan)
            ctx.embed_bwd(d["t"], d["dy"], 1.0, d["g"], count, 5, 4, 1)
            assert np.isnan(d.get("g")).all()
            ctx.embed_bwd(d["t"], d["dy"], 1.0, d["g"], count, 5, 4, 0)
            assert not d.get("g").any()


@pytest.mark.gpu
def test_infinities_and_nans_stay_in_their_row(ctx):
    rng = np.random.default_rng(3)
    count, vocab, cols = 500, 20, 12
    tokens, dy = some_tokens(rng, count, vocab), rng.standard_normal((count, cols)).astype(np.float32)
    bad = tokens[100]
    dy[100] = [np.nan, np.inf, -np.inf] * 4
    want, off = ref.embed_grad(tokens, dy, 1.0, vocab)
    with DeviceArrays(ctx, tokens=ref.device_ints(tokens), dy=dy) as d:
        d.alloc("g", vocab * cols, fill=np.nan)
        ctx.embed_bwd(d["tokens"], d["dy"], 1.0, d["g"], count, vocab, cols)
        got = d.get("g").reshape(vocab, cols)
    assert np.isnan(want[bad]).any() and np.isfinite(np.delete(want, bad, 0)).all()
    ref.assert_near(got, want, np.where(np.isfinite(off), off, 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("count", [700, 20000])
def test_replayed_and_on_other_streams(count):
    from test_captured_calls import capture

    vocab, cols = 300, 48
    rng = np.random.default_rng(count)
    first, second = (some_tokens(rng, count, vocab) for _ in range(2))
    dy = rng.standard_normal((count, cols)).astype(np.float32)
    contexts, results = [cabi.Context(0) for _ in range(2)], []
    try:
        for c in contexts:
            with DeviceArrays(c, t=ref.device_ints(first), dy=dy) as d:
                d.alloc("g", vocab * cols), d.alloc("h", vocab * cols)
                call = lambda out: c.embed_bwd(d["t"], d["dy"], 2.0, d[out], count, vocab, cols)  # noqa: E731
                replay = capture(c, lambda: call("g"))  # (also without a workspace of its size)
                eager = []
                for tokens in (second, first):  # a replay looks at its own tokens
                    c.h2d(d["t"], ref.device_ints(tokens))
                    call("h")
                    replay()
                    eager.append(d.get("h"))
                    assert np.array_equal(d.get("g"), eager[-1])
                assert not np.array_equal(*eager)
                del replay
                results.append(eager[1])
        assert np.array_equal(*results)
    finally:
        for c in contexts:
            c.close()


A, B, C, D = 0x10000, 0x20000, 0x30000, 0x40000  # addresses that nothing reads


@pytest.mark.parametrize("name,why,args", [
    ("embed_fwd", "below", (A, B, 1.0, C, 1 << 31, 4, 4)), ("embed_fwd", "below", (A, B, 1.0, C, 4, 1 << 31, 4)),
    ("embed_fwd", "below", (A, B, 1.0, C, 4, 4, 1 << 30)), ("embed_fwd", "null buffer", (None, B, 1.0, C, 4, 4, 4)),
    ("embed_fwd", "null buffer", (A, None, 1.0, C, 4, 4, 4)), ("embed_fwd", "null buffer", (A, B, 1.0, None, 4, 4, 4)),
    ("embed_fwd", "whole element", (A + 1, B, 1.0, C, 4, 4, 4)), ("embed_fwd", "whole element", (A, B + 2, 1.0, C, 4, 4, 4)),
    ("embed_fwd", "whole element", (A, B, 1.0, C + 3, 4, 4, 4)), ("embed_fwd", "overlaps", (A, B, 1.0, A + 60, 4, 4, 4)),
    ("embed_fwd", "overlaps", (A, B, 1.0, B - 60, 4, 4, 4)),
    ("int8_embed", "null buffer", (None, A, B, 1.0, C, 4, 4, 4)), ("int8_embed", "null buffer", (A, None, B, 1.0, C, 4, 4, 4)),
    ("int8_embed", "null buffer", (A, B, None, 1.0, C, 4, 4, 4)), ("int8_embed", "null buffer", (A, B, C, 1.0, None, 4, 4, 4)),
    ("int8_embed", "16-byte", (A + 4, B, C, 1.0, D, 4, 4, 4)), ("int8_embed", "whole element", (A, B, C, 1.0, D + 2, 4, 4, 4)),
    ("int8_embed", "overlaps", (A, B, C, 1.0, A + 60, 4, 4, 4)), ("int8_embed", "overlaps", (A, B, C, 1.0, B + 12, 4, 4, 4)),
    ("embed_bwd", "below", (A, B, 1.0, C, 1 << 31, 4, 4, 0)), ("embed_bwd", "null buffer", (A, B, 1.0, None, 4, 4, 4, 0)),
    ("embed_bwd", "null buffer", (None, B, 1.0, C, 4, 4, 4, 0)), ("embed_bwd", "null buffer", (A, None, 1.0, C, 4, 4, 4, 0)),
    ("embed_bwd", "overlaps", (A, B, 1.0, B + 60, 4, 4, 4, 0)), ("embed_bwd", "overlaps", (A, B, 1.0, A - 60, 4, 4, 4, 1)),
    ("embed_bwd", "whole element", (A, B, 1.0, C + 2, 4, 4, 4, 1)),
])
def test_refusals(anywhere, name, why, args):  # noqa: F811
    lib = cabi.load()
    call = getattr(lib, "katsu_cuda_" + name)
    assert call(anywhere, *args) == cabi.ERR_INVALID_ARG
    assert why in lib.katsu_cuda_last_error_string().decode()
    assert call(None, *args) == cabi.ERR_INVALID_ARG
    assert "null context" in lib.katsu_cuda_last_error_string().decode()
