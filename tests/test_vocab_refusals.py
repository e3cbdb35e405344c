"""Calls at a language model's two ends that have to be refused: outputs in the place of an input that is not the logits, lists of other
axes than the rows that they are for."""
import numpy as np
import pytest

import katsu_b200 as K
import vocab_ref as ref
from katsu_b200 import cabi
from test_adjust_logits import BASE as LOGITS
from test_adjust_logits import NAMES as LOGITS_NAMES
from test_block_norm import anywhere  # noqa: F401 (fixture)
from test_distill import BASE as DISTILL
from test_distill import NAMES as DISTILL_NAMES


@pytest.mark.parametrize("other", ["teacher", "index", "labels", "weight", "g"])
def test_a_loss_in_place_of_its_logits_and_of_another_input(anywhere, other):  # noqa: F811
    """The gradient may be written where the logits are; a list, a label or a weight that is there too would be overwritten under way."""
    args = {**DISTILL, "dlogits": DISTILL["logits"], other: DISTILL["logits"]}
    lib = cabi.load()
    assert lib.katsu_cuda_distill_bwd(anywhere, *(args[n] for n in DISTILL_NAMES)) == cabi.ERR_INVALID_ARG
    assert "overlaps" in lib.katsu_cuda_last_error_string().decode()


@pytest.mark.parametrize("other", ["history", "prompts", "lengths", "repetition", "presence", "frequency", "bias_tokens", "bias", "allowed"])
def test_logits_adjusted_in_place_and_in_that_of_another_input(anywhere, other):  # noqa: F811
    args = {**LOGITS, "out": LOGITS["logits"], other: LOGITS["logits"]}
    lib = cabi.load()
    assert lib.katsu_cuda_adjust_logits(anywhere, *(args[n] for n in LOGITS_NAMES)) == cabi.ERR_INVALID_ARG
    assert "overlaps" in lib.katsu_cuda_last_error_string().decode()


LISTS = {"history": lambda *shape: {"history": np.zeros(shape, int)},
         "biases": lambda *shape: {"bias_tokens": np.zeros(shape, int), "bias": np.zeros(shape)}}


@pytest.mark.parametrize("of", LISTS.values(), ids=LISTS)
@pytest.mark.parametrize("shape", [(100,), (1, 100), (100, 1), (8, 4), (2, 8), (4,), (4, 3, 2), (2, 2, 3), (1, 4, 5)], ids=str)
def test_lists_that_are_not_a_row_of_logits_each(of, shape):
    """One list for all rows, a transposed one, or more axes: their sizes divide by the rows."""
    with pytest.raises(K.InvalidOperand, match="a list for every row"):
        K.adjust_logits(K.Tensor.zeros([4, 9]), **of(*shape))


@pytest.mark.parametrize("logits,shape", [([9], (2, 3)), ([9], (3, 1)), ([1, 9], (3, 1)), ([1, 9], (1, 1, 3))], ids=str)
def test_lists_of_other_rows_than_the_one(logits, shape):
    for of in LISTS.values():
        with pytest.raises(K.InvalidOperand, match="a list for every row"):
            K.adjust_logits(K.Tensor.zeros(logits), **of(*shape))


@pytest.mark.gpu
@pytest.mark.parametrize("logits", [[50], [1, 50]], ids=str)
@pytest.mark.parametrize("shape", [(7,), (1, 7)], ids=str)
def test_lists_of_one_row(logits, shape):
    rng = np.random.default_rng(2)
    z, history, tokens, bias = (rng.standard_normal(50).astype(np.float32), rng.integers(0, 50, 7), rng.integers(0, 50, 7),
                                rng.standard_normal(7).astype(np.float32))
    got = K.adjust_logits(K.Tensor(z, logits), history.reshape(shape), repetition=1.5, bias_tokens=tokens.reshape(shape), bias=bias.reshape(shape))
    ref.assert_near(got.data(), *ref.adjust(z[None], history[None], None, None, np.float32([1.5]), None, None, tokens[None], bias[None], None))


@pytest.mark.gpu
def test_lists_of_nothing():
    z = np.arange(12, dtype=np.float32)
    for empty in ([], np.zeros((3, 0), int), np.zeros((0, 5), int)):
        got = K.adjust_logits(K.Tensor(z, [3, 4]), history=empty, bias_tokens=empty, bias=empty)
        assert np.array_equal(got.data(), z)


# logits [2, 3, 9] against a teacher [2, 3, 4]: axes whose sizes multiply to the right number, in another order
@pytest.mark.parametrize("what,shape", [("index", (3, 2, 4)), ("index", (4, 6)), ("index", (3, 8)), ("index", (4, 3, 2)), ("index", (6, 2, 2)),
                                        ("index", (8, 3)), ("labels", (3, 2)), ("labels", (1, 3, 1, 2)), ("weight", [3, 2]),
                                        ("weight", [3, 1, 2])], ids=str)
def test_rows_in_another_order(what, shape):
    args = {"teacher": K.Tensor.zeros([2, 3, 4]), "index": np.zeros((2, 3, 4), int)}
    args[what] = K.Tensor.zeros(shape) if what == "weight" else np.zeros(shape, int)
    with pytest.raises(K.InvalidOperand, match=f"{what} must have"):
        K.DistillLoss().forward(K.Tensor.zeros([2, 3, 9]), **args)


@pytest.mark.parametrize("shape", [(4, 6), (8, 3), (12, 2), (4, 3, 2)], ids=str)
def test_lists_of_another_order_than_the_teachers(shape):
    with pytest.raises(K.InvalidOperand, match="index must have"):
        K.DistillLoss().forward(K.Tensor.zeros([6, 9]), K.Tensor.zeros([6, 4]), np.zeros(shape, int))


@pytest.mark.gpu
@pytest.mark.parametrize("index,labels,weight", [((2, 3, 4), (2, 3), [2, 3]), ((6, 4), (6,), [6]), ((24,), (6,), [2, 3, 1]), ((2, 1, 3, 4), (1, 2, 3), [1, 2, 3]), ((2, 12), (2, 3, 1), [1, 6])])
def test_rows_in_order(index, labels, weight):
    """Axes of one value, and axes that are put together, change no order."""
    rng = np.random.default_rng(7)
    z, teacher, at, label = (rng.standard_normal((6, 9)).astype(np.float32), rng.standard_normal((6, 4)).astype(np.float32),
                             rng.integers(-1, 9, (6, 4)), rng.integers(-1, 9, 6))
    w = rng.random(6).astype(np.float32)
    loss = K.DistillLoss(2.0, 0.5, 0.5).forward(K.Tensor(z, [2, 3, 9]), K.Tensor(teacher, [2, 3, 4]), at.reshape(index), label.reshape(labels),
                                               K.Tensor(w, weight))
    assert loss.shape() == [2, 3]
    want, off, _, _ = ref.distill(z, teacher, at, label, w, 2.0, 0.5, 0.5)
    ref.assert_near(loss.data(), want, off)


@pytest.mark.gpu
def test_rows_of_more_axes_than_the_logits():
    """Labels and weights [2, 3] of logits that were made [6, 9] for a product."""
    rng = np.random.default_rng(8)
    z, label, w = rng.standard_normal((6, 9)).astype(np.float32), rng.integers(-1, 9, 6), rng.random(6).astype(np.float32)
    loss = K.DistillLoss(1.0, 0.0, 1.0).forward(K.Tensor(z, [6, 9]), labels=label.reshape(2, 3), weight=K.Tensor(w, [2, 3]))
    want, off, _, _ = ref.distill(z, np.zeros((6, 0)), np.zeros((6, 0), int), label, w, 1.0, 0.0, 1.0)
    ref.assert_near(loss.data(), want, off)
