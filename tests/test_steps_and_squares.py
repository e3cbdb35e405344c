"""A square that nobody has read is not computed before somebody does.  A step of its operand in between must not show in it."""
import numpy as np
import pytest

import katsu_b200 as K

pytestmark = pytest.mark.gpu

V = np.array([1.0, -2.0, 3.0, 0.5], np.float32)


@pytest.fixture(params=[True, False], ids=["fused", "unfused"])
def fusion(request):
    before = K.loss_fusion()
    K.set_loss_fusion(request.param)
    yield
    K.set_loss_fusion(before)


STEPS = {"sgd_step": lambda t: t.sgd_step(0.5), "sgd_step_clipped": lambda t: K.sgd_step_clipped([t], 0.5, 1e9)}


@pytest.mark.parametrize("step", STEPS)
def test_squares_of_what_a_step_changes(fusion, step):
    w = K.Tensor(V, [4])
    first = w.mul(w)
    view = w.reshape([2, 2])
    of_view, again = view.mul(view), first.mul(first)
    penalty = w.mul(w).sum()
    w.mul(K.Tensor(np.ones(4, np.float32), [4])).sum().backward()
    STEPS[step](w)
    assert np.array_equal(w.data(), V - 0.5)
    assert np.array_equal(first.data(), V * V) and np.array_equal(of_view.data(), V * V) and np.array_equal(again.data(), (V * V) * (V * V))
    assert np.array_equal(penalty.parents()[0].data(), V * V)
    later = w.mul(w)
    STEPS[step](w)
    assert np.array_equal(later.data(), (V - 0.5) * (V - 0.5)) and np.array_equal(w.data(), V - 1)
    assert np.array_equal(w.mul(w).data(), (V - 1) * (V - 1))


@pytest.mark.parametrize("step", STEPS)
def test_squares_of_a_view_that_is_stepped(fusion, step):
    w = K.Tensor(V, [4])
    square, view = w.mul(w), w.reshape([2, 2])
    view.mul(K.Tensor(np.ones(4, np.float32), [2, 2])).sum().backward()
    STEPS[step](view)
    assert np.array_equal(square.data(), V * V)
