"""Tables, rows and logits of more than 2^32 values, and vocabularies near 2^31: the operators on a few rows at the far end give what
they give on these rows alone."""
import numpy as np
import pytest

import vocab_ref as ref
from parity_util import DeviceArrays

pytestmark = pytest.mark.gpu


def put(ctx, address, at, values):
    """`values` from element `at` of the buffer on."""
    ctx.h2d(address + 4 * at, np.ascontiguousarray(values, np.float32).reshape(-1))
    ctx.sync()


def get(ctx, address, at, shape):
    return ctx.download(address + 4 * at, int(np.prod(shape))).reshape(shape)


@pytest.mark.parametrize("cols", [4200, 4201])
def test_a_table_of_more_than_2_to_the_32_values(ctx, cols):
    vocab, rng = (1 << 20) + 77, np.random.default_rng(cols)
    tokens = np.array([vocab - 1, 3, vocab - 2, vocab - 1, vocab // 2, -1, 3] * 50)
    rows = np.unique(tokens[tokens >= 0])
    table, dy = rng.standard_normal((len(rows), cols)).astype(np.float32), rng.standard_normal((len(tokens), cols)).astype(np.float32)
    small = np.searchsorted(rows, tokens)
    small[tokens < 0] = -1
    with DeviceArrays(ctx, t=ref.device_ints(tokens), dy=dy) as d:
        d.alloc("table", vocab * cols), d.alloc("y", len(tokens) * cols)
        for row, values in zip(rows, table):
            put(ctx, d["table"], int(row) * cols, values)
        ctx.embed_fwd(d["table"], d["t"], 2.0, d["y"], len(tokens), vocab, cols)
        assert np.array_equal(d.get("y").reshape(dy.shape), ref.embed(table, small, 2.0).astype(np.float32))
        want, off = ref.embed_grad(small, dy, 0.5, len(rows))
        for accumulate in (1, 0):
            ctx.embed_bwd(d["t"], d["dy"], 0.5, d["table"], len(tokens), vocab, cols, accumulate)
            for i, row in enumerate(rows):
                before = table[i].astype(np.float64) * accumulate
                ref.assert_near(get(ctx, d["table"], int(row) * cols, (cols,)), want[i] + before, off[i] + 2 * ref.U * (np.abs(before) + np.abs(want[i])))
            for row in (0, vocab // 2 + 1, vocab - 3):
                assert not get(ctx, d["table"], row * cols, (cols,)).any()


@pytest.mark.parametrize("cols", [4096, 4099])
def test_more_than_2_to_the_32_values_looked_up(ctx, cols):
    """And their gradient: more rows of it than 2^32 values."""
    count, vocab, rng = (1 << 20) + 130, 9, np.random.default_rng(cols)
    table = rng.standard_normal((vocab, cols)).astype(np.float32)
    tokens = rng.integers(-1, vocab, count)
    with DeviceArrays(ctx, t=ref.device_ints(tokens), table=table) as d:
        d.alloc("y", count * cols)
        ctx.embed_fwd(d["table"], d["t"], 1.5, d["y"], count, vocab, cols)
        for lo in (0, count // 2, count - 5):
            assert np.array_equal(get(ctx, d["y"], lo * cols, (5, cols)), ref.embed(table, tokens[lo: lo + 5], 1.5).astype(np.float32))
        ctx.embed_bwd(d["t"], d["y"], 1.0, d["table"], count, vocab, cols)
        got = d.get("table").reshape(vocab, cols)
    # every value of a token is the same number: the sum is the count's multiple, off by its additions
    number = np.bincount(tokens[tokens >= 0], minlength=vocab).astype(np.float64)
    want = number[:, None] * (table * np.float32(1.5)).astype(np.float64)
    assert (np.abs(got - want) <= ref.U * (64 + 32 + number / 2048 + 40)[:, None] * np.abs(want)).all()


def test_a_vocabulary_of_more_than_2_to_the_30_tokens(ctx):
    """Keys of 31 bits: four passes of the sort."""
    vocab, count, rng = (1 << 30) + 9, 9000, np.random.default_rng(1)
    rows = np.sort(np.unique(np.concatenate([rng.integers(0, vocab, 3000), [0, vocab - 1]])))
    small = rng.integers(-1, len(rows), count)
    tokens = np.where(small < 0, -1, rows[small])
    tokens[:2] = vocab, 2 ** 31 - 1
    small[:2] = -1
    dy = rng.standard_normal((count, 1)).astype(np.float32)
    want, off = ref.embed_grad(small, dy, 1.0, len(rows))
    with DeviceArrays(ctx, t=ref.device_ints(tokens), dy=dy) as d:
        d.alloc("g", vocab)
        ctx.embed_bwd(d["t"], d["dy"], 1.0, d["g"], count, vocab, 1, 1)
        got = np.array([get(ctx, d["g"], int(r), (1,)) for r in rows[::37]])
        ref.assert_near(got, want[::37], off[::37])
        ctx.call("katsu_cuda_sum", d["g"], d["dy"], vocab)  # nothing anywhere else
        assert abs(d.get("dy")[0] - want.sum()) <= 1e-3


@pytest.mark.parametrize("vocab", [131072, 131075])
def test_more_than_2_to_the_32_logits(ctx, vocab):
    rows, top, rng = (1 << 15) + 11, 3, np.random.default_rng(vocab)
    last = 4
    z, teacher = rng.standard_normal((last, vocab)).astype(np.float32), rng.standard_normal((last, top)).astype(np.float32)
    index, labels, weight = rng.integers(0, vocab, (last, top)), rng.integers(0, vocab, last), np.zeros(rows, np.float32)
    weight[-last:] = 1  # the rows in front are not read
    lo = rows - last
    full = lambda v, fill: np.concatenate([np.full((lo, *v.shape[1:]), fill), v])  # noqa: E731
    with DeviceArrays(ctx, t=full(teacher, 0.0), i=ref.device_ints(full(index, -1)), l=ref.device_ints(full(labels, -1)), w=weight) as d:
        d.alloc("z", rows * vocab), d.alloc("loss", rows, fill=np.nan)
        put(ctx, d["z"], lo * vocab, z)
        put(ctx, d["z"], (lo - 1) * vocab, np.full(vocab, np.nan))
        common = (d["z"], d["t"], d["i"], d["l"], d["w"], 2.0, 0.5, 0.5)
        want, off, dz, doff = ref.distill(z, teacher, index, labels, None, 2.0, 0.5, 0.5)
        ctx.distill_fwd(*common, d["loss"], rows, vocab, top)
        loss = d.get("loss")
        assert not loss[:lo].any()
        ref.assert_near(loss[lo:], want, off)
        # in place, as there is no memory to waste
        ctx.distill_bwd(*common, None, d["loss"], d["z"], rows, vocab, top)
        ref.assert_near(d.get("loss")[lo:], want, off)
        ref.assert_near(get(ctx, d["z"], lo * vocab, (last, vocab)), dz, doff)
        assert not get(ctx, d["z"], (lo - 1) * vocab, (vocab,)).any()
        # logits of a served model, at the same places
        put(ctx, d["z"], lo * vocab, z)
        history, words = rng.integers(0, vocab, (last, 6)), rng.random((last, vocab)) < 0.5
        all_words = full(ref.words_of(words), -1)
        rep = np.full(rows, 1.5, np.float32)
        bias_tokens, bias = rng.integers(0, vocab, (last, 2)), rng.standard_normal((last, 2)).astype(np.float32)
        with DeviceArrays(ctx, h=ref.device_ints(full(history, -1)), m=ref.device_ints(all_words), rep=rep,
                          bt=ref.device_ints(full(bias_tokens, -1)), b=full(bias, 0.0)) as e:
            ctx.adjust_logits(d["z"], e["h"], None, None, e["rep"], None, None, e["bt"], e["b"], e["m"], d["z"], rows, vocab, 6, 2)
        want, off = ref.adjust(z, history, None, None, rep[-last:], None, None, bias_tokens, bias, words)
        ref.assert_near(get(ctx, d["z"], lo * vocab, (last, vocab)), want, off)


def test_long_histories_of_many_rows(ctx):
    """2^15 tokens and more are counted in 32 bits, in slices of the largest size."""
    rows, vocab, cols, rng = 600, 17001, 1 << 15, np.random.default_rng(3)
    history = rng.integers(0, 40, (rows, cols))
    history[:, 1::2] = rng.integers(0, vocab, (rows, cols // 2))
    z, f = rng.standard_normal((rows, vocab)).astype(np.float32), np.full(rows, 0.01, np.float32)
    lengths = rng.integers(0, cols + 1, rows)
    lengths[-1] = cols
    with DeviceArrays(ctx, z=z, h=ref.device_ints(history), l=ref.device_ints(lengths), f=f) as d:
        d.alloc("out", z.size, fill=np.nan)
        ctx.adjust_logits(d["z"], d["h"], None, d["l"], None, None, d["f"], None, None, None, d["out"], rows, vocab, cols, 0)
        got = d.get("out").reshape(rows, vocab)
    few = [0, 1, 299, rows - 1]
    ref.assert_near(got[few], *ref.adjust(z[few], history[few], None, lengths[few], None, None, f[few], np.zeros((4, 0)), None, None))
