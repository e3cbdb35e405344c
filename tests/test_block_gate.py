"""How BlockNorm reads a gate's shape: its rows go to runs of x's rows, and a shape that broadcasting would read otherwise is refused."""
import numpy as np
import pytest

import block_ref
import katsu_b200 as K
from parity_util import rel_l2

TOL = 1e-5  # chains of a few f32 operations


def tensor(a):
    return K.Tensor(a, list(a.shape))


# x's shape, the gate's, and the gate as it stands before every row by the documented reading
TAKEN = [
    ([6, 8], [8]), ([6, 8], [1, 8]), ([6, 8], [3, 8]), ([6, 8], [6, 8]), ([2, 3, 8], [2, 8]), ([2, 3, 8], [2, 1, 8]), ([2, 3, 8], [2, 3, 8]),
    ([2, 3, 4, 8], [6, 8]), ([2, 3, 4, 8], [2, 3, 8]), ([2, 3, 4, 8], [2, 3, 1, 8]), ([2, 3, 4, 8], [1, 1, 1, 8]), ([1, 4, 8], [4, 8]),
    ([4, 1, 8], [4, 8]), ([4, 4, 8], [4, 8]), ([4, 8], [1, 4, 8]), ([1, 4, 1, 8], [4, 1, 8]), ([2, 3, 4, 8], [12, 8]),
]
REFUSED = [
    ([2, 3, 4, 8], [4, 8]), ([2, 3, 4, 8], [3, 1, 8]), ([2, 3, 4, 8], [3, 4, 8]), ([3, 4, 8], [1, 4, 8]), ([3, 4, 8], [4, 8]),
    ([2, 2, 4, 8], [4, 8]), ([2, 3, 4, 8], [2, 1, 4, 8]), ([2, 3, 4, 8], [1, 3, 1, 8]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,gate_shape", TAKEN, ids=str)
def test_runs_of_rows(shape, gate_shape):
    rng = np.random.default_rng([len(shape), *gate_shape])
    x, h, c = (rng.standard_normal(shape).astype(np.float32) for _ in range(3))
    gate, w = rng.standard_normal(gate_shape).astype(np.float32), rng.standard_normal(8).astype(np.float32)
    t = [tensor(v) for v in (x, h, gate)]
    r, n = K.BlockNorm(None, K.Norm(tensor(w), eps=1e-5)).forward(*t)
    n.mul(tensor(c)).sum().backward()
    flat = lambda v: v.reshape(-1, 8)  # noqa: E731
    r64, n64 = block_ref.forward(flat(x), flat(h), flat(gate), None, None, w, None, 1.0, 1e-5, False)
    want = block_ref.backward(r64, flat(h), flat(gate), None, None, w, 1.0, 1e-5, False, None, flat(c))
    assert rel_l2(r.data(), r64) <= TOL and rel_l2(n.data(), n64) <= TOL
    for tensor_of, name in zip(t, ("dx", "dh", "dgate")):
        assert rel_l2(tensor_of.grad(), want[name]) <= TOL, name


@pytest.mark.parametrize("shape,gate_shape", REFUSED, ids=str)
def test_shapes_that_broadcasting_reads_otherwise(shape, gate_shape):
    x, gate, w = (tensor(np.ones(s, np.float32)) for s in (shape, gate_shape, [8]))
    with pytest.raises(K.InvalidOperand, match="axes"):
        K.BlockNorm(K.Norm(w)).forward(x, x, gate)
