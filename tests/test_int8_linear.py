"""Int8Linear holds the layer as it was when it was made."""
import numpy as np
import pytest

import katsu_b200 as K


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 40])
def test_later_steps_change_neither_weights_nor_bias(m):
    rng = np.random.default_rng(m)
    x, w, b = (rng.standard_normal(s).astype(np.float32) for s in ((m, 48), (48, 24), (24,)))
    xt, wt, bt = (K.Tensor(v, list(v.shape)) for v in (x, w, b))
    served = K.Int8Linear(wt, bt)
    before = served.forward(xt).data().copy()
    assert np.array_equal(before, (K.Int8Linear(wt).forward(xt).data().reshape(m, 24) + b).reshape(-1))
    wt.mul(wt).sum().add(bt.mul(bt).sum()).backward()
    K.sgd_step_clipped([wt, bt], 0.25, 1.0)
    assert not np.array_equal(bt.data(), b) and not np.array_equal(wt.data(), w.reshape(-1))
    assert np.array_equal(served.forward(xt).data(), before)
    del bt, wt
    assert np.array_equal(served.forward(xt).data(), before)
