"""The gradient of a table of small whole numbers: every sum of them is a number of f32, whatever the order, so that the kernels have to
give the sums themselves.  One token that is left out, taken twice or added to another row shows."""
import numpy as np
import pytest

import vocab_ref as ref
from parity_util import DeviceArrays
from test_embed import some_tokens


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


def check(ctx, count, vocab, cols, how, accumulate, shift=0, seed=0):
    """Twice, as what threads write at the same time need not come out alike."""
    rng = np.random.default_rng([seed, count, vocab, cols])
    tokens, dy, before = some_tokens(rng, count, vocab, how), whole_numbers(rng, (count, cols)), whole_numbers(rng, (vocab, cols))
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
