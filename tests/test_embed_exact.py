"""The gradient of a table of small whole numbers: every sum of them is a number of f32, whatever the order, so that the kernels have to
give the sums themselves.  One token that is left out, taken twice or added to another row shows."""
import numpy as np
import pytest

import vocab_ref as ref
from parity_util import DeviceArrays
from test_embed import GRADS, some_tokens


def whole_numbers(rng, shape):
    """-3 to 3, and never 0."""
    return (rng.integers(1, 4, shape) * rng.choice([-1, 1], shape)).astype(np.float32)


def sums_of(tokens, dy, vocab):
    """[vocab, cols]: the sums of every token's rows."""
    there = ref.valid(tokens, vocab)
    order = np.argsort(tokens[there], kind="stable")
    rows, keys = dy[there][order].astype(np.int64), tokens[there][order]
    want = np.zeros((vocab, dy.shape[1]), np.int64)
    if len(keys):
        starts = np.flatnonzero(np.r_[True, keys[1:] != keys[:-1]])
        want[keys[starts]] = np.add.reduceat(rows, starts, 0)
    return want


def check(ctx, count, vocab, cols, how, accumulate, shift=0):
    rng = np.random.default_rng([count, vocab, cols])
    check_tokens(ctx, some_tokens(rng, count, vocab, how), vocab, cols, rng, accumulate, shift)


def check_tokens(ctx, tokens, vocab, cols, rng, accumulate=1, shift=0):
    """Twice, as what threads write at the same time need not come out alike."""
    count, dy, before = len(tokens), whole_numbers(rng, (len(tokens), cols)), whole_numbers(rng, (vocab, cols))
    want = sums_of(tokens, dy, vocab) * 0.5 + (before if accumulate else 0)
    assert np.abs(want).max() + 3 < 2 ** 22  # (halves of numbers below 2^24 are numbers of f32)
    edge = np.full(4, 7.0, np.float32)
    start = before if accumulate else np.full((vocab, cols), np.nan, np.float32)
    with DeviceArrays(ctx, tokens=ref.device_ints(tokens), dy=np.concatenate([edge[:shift], dy.reshape(-1)])) as d:
        for name in ("first", "second"):
            d.ptr[name] = ctx.upload(np.concatenate([edge[:shift], start.reshape(-1), edge]))
            d.size[name] = shift + vocab * cols + 4
            ctx.embed_bwd(d["tokens"], d["dy"] + 4 * shift, 0.5, d[name] + 4 * shift, count, vocab, cols, accumulate)
            got = d.get(name)
            assert (got[:shift] == 7).all() and (got[shift + vocab * cols:] == 7).all()
            wrong = np.argwhere(got[shift: shift + vocab * cols].reshape(vocab, cols) != want)
            assert len(wrong) == 0, (len(wrong), wrong[:5])


# Rows that are whole 16-byte units have groups of half as many threads as others of their width: the fold of a run has a warp for both.
@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("count,vocab,how", [(3000, 3, "half"), (9000, 2, "one"), (40000, 5, "half"), (30000, 700, "zipf")])
@pytest.mark.parametrize("cols", [4, 8, 12, 16, 20, 28, 32, 33, 36, 40, 44, 48, 52, 56, 60, 63, 64, 65, 68, 128])
def test_runs_over_many_pieces_in_narrow_rows(ctx, cols, count, vocab, how, shift, accumulate):
    check(ctx, count, vocab, cols, how, accumulate, shift)


# Counts on both sides of those where the gradient takes another way, runs of many pieces, bundles and parts among them
@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("count,vocab,cols,how", GRADS + [
    (1000003, 7, 4, "half"), (400000, 3, 17, "one"), (400000, 40, 64, "blocks"), (131072, 1, 130, "one"), (262144, 16, 16, "blocks"), (50000, 9, 40, "half")])
def test_every_sum(ctx, count, vocab, cols, how, accumulate):
    check(ctx, count, vocab, cols, how, accumulate)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [4, 12, 24, 48, 64, 200])
@pytest.mark.parametrize("off", [-1, 0, 1])
@pytest.mark.parametrize("piece", [8, 16, 32])
def test_runs_that_end_around_pieces_and_bundles(ctx, piece, off, cols):
    """Runs of 1, 2, 31 to 33 and 64 pieces behind each other, a token more or less than whole ones."""
    lengths = [max(1, piece * n + off) for n in (1, 2, 31, 32, 33, 64, 1, 0, 96, 5)]
    tokens = np.repeat(np.arange(len(lengths)), lengths)
    for start in (0, 1, 7):  # what is no token sorts behind; a token in front moves all ends
        keys = np.concatenate([np.zeros(start, int), tokens + 1])
        rng = np.random.default_rng([piece, cols, start])
        order = rng.permutation(len(keys))
        for times in (1, 9):  # (longer lists have longer pieces)
            check_tokens(ctx, np.tile(keys[order], times), len(lengths) + 1, cols, rng)
