"""The loss and its gradient on both sides of the sizes where blocks get other numbers of threads, and rows other numbers of blocks."""
import numpy as np
import pytest

import vocab_ref as ref
from test_distill import inputs, run

MANY = 2400  # rows: more than sixteen for each of 148 SMs


class Formula:
    """A case's loss and gradient in 64 bits, with what f32 may be off them."""

    def __init__(self, a, T, soft, hard):
        self.a, self.how = a, (T, soft, hard)
        self.loss, self.off, self.dz, self.doff = ref.distill(a["z"], a["teacher"], a["index"], a["labels"], a["weight"], T, soft, hard, a["g"])
        listed = np.zeros(a["z"].shape)
        there = ref.valid(a["index"], a["z"].shape[1])
        np.add.at(listed, (np.nonzero(there)[0], a["index"][there]), 1.0)
        # a token's probability is a sum of as many roundings as it is listed times, of at most 1
        self.doff += np.abs(a["g"] * a["weight"])[:, None] * soft * T * ref.U * listed

    def check(self, ctx, **more):
        fwd, bwd, got = run(ctx, self.a, *self.how, **more)
        ref.assert_near(fwd, self.loss, self.off, "loss")
        ref.assert_near(bwd, self.loss, self.off, "loss beside the gradient")
        dz, doff = self.dz, self.doff
        if more.get("accumulate") is not None:
            before = more["accumulate"].astype(np.float64)
            # added to twice at listed tokens: the row's part, then the list's
            dz, doff = dz + before, doff + 2 * ref.U * (np.abs(before) + np.abs(dz)) + 2 * ref.U * np.abs(dz + before)
        ref.assert_near(got, dz, doff, "gradient")
        return got


# 64 threads for many short rows, 128 for few and for longer ones (4 x 1024 values are the border), lists on both sides of 256 entries
@pytest.mark.gpu
@pytest.mark.parametrize("T,soft,hard", [(1.0, 0.7, 0.3), (2.0, 0.5, 0.5)])
@pytest.mark.parametrize("rows,vocab,top", [(MANY, 10, 3), (MANY, 50, 5), (MANY, 50, 300), (MANY, 1003, 5), (40, 1003, 5), (MANY, 1003, 300), (MANY, 4096, 5),
                                            (MANY, 4097, 5), (MANY, 4100, 5), (40, 4096, 300), (2, 50, 300)])
def test_short_rows(ctx, rows, vocab, top, T, soft, hard):
    want = Formula(inputs(rows, vocab, top), T, soft, hard)
    assert np.array_equal(want.check(ctx), want.check(ctx, in_place=True))
    want.check(ctx, shift=1, out_shift=1)
    want.check(ctx, shift=3, out_shift=2, accumulate=np.random.default_rng(5).standard_normal((rows, vocab)).astype(np.float32))


# 128 and 256 threads, 256 and 512 for a gradient, one and more blocks to a row by its length and by the number of rows
@pytest.mark.gpu
@pytest.mark.parametrize("T,soft,hard", [(1.0, 1.0, 0.0), (2.0, 0.5, 0.5)])
@pytest.mark.parametrize("rows,vocab,top", [(20, 8192, 5), (20, 8193, 257), (20, 16384, 256), (20, 16388, 257), (700, 16388, 5), (320, 32768, 20), (320, 32772, 20),
                                            (40, 65540, 5), (37, 65536, 300)])
def test_long_rows(ctx, rows, vocab, top, T, soft, hard):
    want = Formula(inputs(rows, vocab, top), T, soft, hard)
    assert np.array_equal(want.check(ctx), want.check(ctx, in_place=True))


@pytest.mark.gpu
@pytest.mark.parametrize("T,soft,hard", [(1.0, 0.0, 1.0), (1.0, 0.5, 0.5), (2.0, 0.5, 1.0), (0.5, 1.0, 0.3)])
@pytest.mark.parametrize("vocab", [2, 50, 1003, 40001])
def test_logits_that_are_large_and_alike(ctx, vocab, T, soft, hard):
    """Rows of one number, a mask's lowest one among them, and rows of a few numbers far from 0: the loss is that of their differences."""
    a = inputs(12, vocab, 4)
    low = np.finfo(np.float32).min
    for row, value in enumerate([low, -1e30, 1e30, -low, 3e20, -2.0 ** 60, low, 1e9]):
        a["z"][row] = value
    a["z"][8] = np.where(np.arange(vocab) % 2, 1e30, low)           # half of them masked, the others alike
    a["z"][9] = 2.0 ** 40 + 2.0 ** 18 * (np.arange(vocab) % 3)      # steps of the numbers there
    a["z"][10] = -2.0 ** 26 + 4.0 * (np.arange(vocab) % 5)
    a["index"][8], a["labels"][8] = 1, 1
    a["labels"][:8] = np.arange(8) % vocab
    a["weight"][:], a["teacher"] = 1.0, np.random.default_rng(1).standard_normal(a["teacher"].shape).astype(np.float32)
    Formula(a, T, soft, hard).check(ctx)
