"""Norm, BlockNorm, Int8Linear, clipping and the clipped step on the graph, alone and together as a training step uses them."""
import numpy as np
import pytest

import block_ref
import katsu_b200 as K
from parity_util import rel_l2

pytestmark = pytest.mark.gpu

# f32 chains of a few operations over rows of up to 96 values; products in 3xTF32 mode hold 1e-5 by their documents
TOL = 1e-5


def f(rng, *shape, mean=0.0, std=1.0):
    return (mean + std * rng.standard_normal(shape)).astype(np.float32)


def tensor(a):
    return K.Tensor(a, list(a.shape))


def grad(t, shape=None):
    g = t.grad()
    return None if g is None else g.reshape(shape or t.shape())


def make(seed, rows, cols, gate_rows, layer):
    rng = np.random.default_rng(seed)
    a = {"x": f(rng, rows, cols), "h": f(rng, rows, cols), "gate": f(rng, gate_rows, cols, mean=1.0) if gate_rows else None}
    for name in ("post", "pre"):
        a[name + "_w"] = f(rng, cols, mean=1.0, std=0.2)
        a[name + "_b"] = f(rng, cols) if layer else None
    return a, {k: None if v is None else tensor(v) for k, v in a.items()}


def layers(t, layer, scale=0.5, eps=1e-5, post=True, pre=True):
    norm = lambda name: K.Norm(t[name + "_w"], t[name + "_b"], eps=eps, layer=layer)  # noqa: E731
    return K.BlockNorm(norm("post") if post else None, norm("pre") if pre else None, scale)


@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("gate_rows", [0, 1, 4, 12])
@pytest.mark.parametrize("also_r", [False, True])
def test_block(layer, gate_rows, also_r):
    """loss = sum(n c) (+ sum(r d)): the norm's part goes into the sum's pass, with and without another gradient of r."""
    rows, cols = 12, 40
    a, t = make(1, rows, cols, gate_rows, layer)
    rng = np.random.default_rng(2)
    c, e = f(rng, rows, cols), f(rng, rows, cols)
    r, n = layers(t, layer).forward(t["x"], t["h"], t["gate"])
    loss = n.mul(tensor(c)).sum()
    if also_r:
        loss = loss.add(r.mul(tensor(e)).sum())
    loss.backward()
    args = [a[k] for k in ("gate", "post_w", "post_b", "pre_w")]
    r64, n64 = block_ref.forward(a["x"], a["h"], *args, a["pre_b"], 0.5, 1e-5, layer)
    assert rel_l2(r.data(), r64) <= TOL and rel_l2(n.data(), n64) <= TOL
    want = block_ref.backward(r64, a["h"], *args, 0.5, 1e-5, layer, e if also_r else None, c)
    for name, v in want.items():
        tensor_of = t[name[1:]]
        if tensor_of is not None:
            assert rel_l2(grad(tensor_of), v) <= TOL, name
    assert rel_l2(grad(r), want["dx"]) <= TOL  # the gradient of the node between is all of it
    assert rel_l2(grad(n), c) == 0
    op = r.op()
    assert (op.kind, op.scale, op.layer, op.gate, op.post, op.bias) == ("BlockSum", 0.5, layer, bool(gate_rows), True, layer)
    assert n.op().kind == "Norm" and n.parents()[0].id() == r.id()


def evaluate(build, names, a):
    """Gradients of build(tensors).sum-like scalar, and the same by central differences of its 64-bit twin along random ways."""
    t = {k: tensor(v) for k, v in a.items()}
    build(K_GRAPH, t).backward()
    return {k: grad(t[k]) for k in names}


class K_GRAPH:
    """The operations on device tensors."""

    add, mul, matmul = K.Tensor.add, K.Tensor.mul, K.Tensor.matmul
    total = K.Tensor.sum

    @staticmethod
    def norm(x, w):
        return K.Norm(w, eps=1e-3).forward(x)

    @staticmethod
    def block(x, h, gate, post, pre):
        return K.BlockNorm(K.Norm(post, eps=1e-3), K.Norm(pre, eps=1e-3), 0.7).forward(x, h, gate)


class NUMPY:
    """The same in 64 bits."""

    add, mul, matmul, total = (staticmethod(v) for v in (np.add, np.multiply, np.matmul, np.sum))

    @staticmethod
    def norm(x, w):
        return block_ref.norm(x, w, None, 1e-3, False)

    @staticmethod
    def block(x, h, gate, post, pre):
        gate = None if gate is None else np.atleast_2d(gate)
        return block_ref.forward(x, h, gate, post, None, pre, None, 0.7, 1e-3, False)


def two_blocks(o, t):
    """Two blocks of one stream; the second norm's weights are shared, h2 is used twice, x is added again at the end."""
    n0 = o.norm(t["x"], t["w0"])
    h1 = o.matmul(n0, t["m1"])
    r1, n1 = o.block(t["x"], h1, t["gate"], t["w1"], t["w2"])
    h2 = o.matmul(n1, t["m2"])
    r2, n2 = o.block(r1, h2, None, t["w2"], t["w2"])
    return o.total(o.mul(o.add(o.add(n2, r2), o.mul(h2, t["x"])), t["c"]))


def same_tensor_twice(o, t):
    """x is the block's output as well; one weight in both norms."""
    r, n = o.block(t["x"], t["x"], t["x"], t["w1"], t["w1"])
    return o.total(o.add(o.mul(n, t["c"]), o.mul(r, n)))


def computed_weight(o, t):
    """A weight that is no leaf: its gradient travels on."""
    r, n = o.block(t["x"], t["c"], t["gate"], t["w1"], o.mul(t["w1"], t["w2"]))
    return o.total(o.mul(n, o.mul(n, t["c"])))


def norm_of_a_sum_twice(o, t):
    """Two norms of one residual stream: one goes into the sum's pass, the other comes before it."""
    r, n = o.block(t["x"], t["c"], t["gate"], t["w1"], t["w2"])
    return o.total(o.mul(o.mul(o.norm(r, t["w0"]), n), t["c"]))


@pytest.mark.parametrize("build", [two_blocks, same_tensor_twice, computed_weight, norm_of_a_sum_twice])
def test_graphs_against_differences(build):
    rows, cols = 10, 24
    rng = np.random.default_rng(3)
    a = {"x": f(rng, rows, cols), "c": f(rng, rows, cols), "gate": f(rng, cols, mean=1.0, std=0.3)}
    a.update({k: f(rng, cols, mean=1.0, std=0.2) for k in ("w0", "w1", "w2")})
    a.update({k: f(rng, cols, cols, std=0.2) for k in ("m1", "m2")})
    t = {k: tensor(v) for k, v in a.items()}
    loss = build(K_GRAPH, t)
    loss.backward()
    exact = {k: v.astype(np.float64) for k, v in a.items()}
    value = float(build(NUMPY, exact))
    # a sum of 240 values of magnitude up to a few, after chains that hold TOL
    assert abs(loss.data()[0] - value) <= 240 * 10 * TOL
    for k in a:
        g = grad(t[k])
        if g is None:
            continue
        way, step = rng.standard_normal(a[k].shape), 1e-5
        ends = [float(build(NUMPY, dict(exact, **{k: exact[k] + s * step * way}))) for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * step)
        assert abs((g * way).sum() - slope) <= 1e-4 * (np.abs(g * way).sum() + 1e-3), k


def test_gradients_accumulate_and_are_checked_before():
    a, t = make(4, 6, 32, 1, False)
    layer = layers(t, False)
    for _ in range(2):
        r, n = layer.forward(t["x"], t["h"], t["gate"])
        n.mul(n).sum().backward()
    r64, n64 = block_ref.forward(*(a[k] for k in ("x", "h", "gate", "post_w", "post_b", "pre_w", "pre_b")), 0.5, 1e-5, False)
    want = block_ref.backward(r64, *(a[k] for k in ("h", "gate", "post_w", "post_b", "pre_w")), 0.5, 1e-5, False, None, 2 * n64)
    for name in ("dx", "dh", "dgate", "dpost_w", "dpre_w"):
        assert rel_l2(grad(t[name[1:]]), 2 * want[name]) <= TOL, name
    with t["x"].borrow_grad():
        with pytest.raises(K.GradientBorrowed):
            n.mul(n).sum().backward()


def test_shapes_of_more_axes_and_none():
    rng = np.random.default_rng(5)
    x, h, w = f(rng, 2, 3, 4, 8), f(rng, 2, 3, 4, 8), f(rng, 8)
    gate = f(rng, 2, 1, 8)
    r, n = K.BlockNorm(None, K.Norm(tensor(w), eps=1e-5)).forward(tensor(x), tensor(h), tensor(gate))
    r64, n64 = block_ref.forward(x.reshape(24, 8), h.reshape(24, 8), gate.reshape(2, 8), None, None, w, None, 1.0, 1e-5, False)
    assert r.shape() == [2, 3, 4, 8] and n.shape() == [2, 3, 4, 8]
    assert rel_l2(r.data(), r64) <= TOL and rel_l2(n.data(), n64) <= TOL
    r, n = K.BlockNorm().forward(tensor(x), tensor(h))
    assert n is None and rel_l2(r.data(), x + h) <= TOL
    # no rows: nothing to do, and gradients of zeros
    e, wt = K.Tensor.zeros([0, 8]), tensor(w)
    r, n = K.BlockNorm(K.Norm(wt), K.Norm(wt)).forward(e, K.Tensor.zeros([0, 8]))
    assert n.shape() == [0, 8]
    n.sum().backward()
    assert not grad(wt).any() and grad(e).size == 0


def test_refusals():
    rng = np.random.default_rng(6)
    x, w = tensor(f(rng, 4, 8)), tensor(f(rng, 8))
    norm = K.Norm(w)
    for call in (lambda: K.Norm(x), lambda: K.Norm(w, x), lambda: K.Norm(w, eps=-1.0), lambda: K.Norm(w, eps=float("nan")),
                 lambda: norm.forward(tensor(f(rng, 4, 7))), lambda: norm.forward(K.Tensor.zeros([])),
                 lambda: norm.forward(K.Tensor.zeros([3, 0])), lambda: K.BlockNorm(norm, K.Norm(w, eps=1e-3)),
                 lambda: K.BlockNorm(norm, K.Norm(w, layer=True)), lambda: K.BlockNorm(norm).forward(x, x, tensor(f(rng, 3, 8))),
                 lambda: K.BlockNorm(norm).forward(x, x, tensor(f(rng, 4))), lambda: K.Int8Linear(x, x),
                 lambda: K.Int8Linear(K.Tensor.zeros([0, 4])), lambda: K.Int8Linear(K.Tensor.zeros([133145, 1])),
                 lambda: K.clip_grad_norm([x], -1.0), lambda: K.sgd_step_clipped([x], 0.1, float("nan"))):
        with pytest.raises(K.InvalidOperand):
            call()
    with pytest.raises(K.ShapeMismatch):
        K.BlockNorm(norm).forward(x, tensor(f(rng, 8, 4)))
    with pytest.raises(K.RankMismatch):
        K.Int8Linear(w)
    with pytest.raises(K.RankMismatch):
        K.Int8Linear(x).forward(w)
    with pytest.raises(K.MatmulMismatch) as e:
        K.Int8Linear(x).forward(x)
    assert (e.value.left_columns, e.value.right_rows) == (8, 4)
    for call in (lambda: K.grad_norm([x]), lambda: K.clip_grad_norm([x], 1.0), lambda: K.sgd_step_clipped([x], 0.1, 1.0)):
        with pytest.raises(K.DeviceError):
            call()
    x.mul(x).sum().backward()
    for call in (lambda: K.grad_norm([x, x]), lambda: K.clip_grad_norm([x, x], 1.0), lambda: K.sgd_step_clipped([x, x.clone()], 0.1, 1.0)):
        with pytest.raises(K.InvalidOperand):
            call()
    with x.borrow_grad():
        for call in (lambda: K.clip_grad_norm([x], 1.0), lambda: K.sgd_step_clipped([x], 0.1, 1.0)):
            with pytest.raises(K.GradientBorrowed):
                call()


def test_clipping_leaves_gradients_that_share_a_buffer_apart():
    """a + b hands both the same gradient; clipping a's must not change b's, and a symbolic gradient is written out."""
    rng = np.random.default_rng(7)
    a, b, c = tensor(f(rng, 50)), tensor(f(rng, 50)), tensor(f(rng, 50))
    a.add(b).mul(c).sum().backward()
    before, other = grad(a).copy(), grad(b).copy()
    norm = np.linalg.norm(before.astype(np.float64))
    got = K.clip_grad_norm([a], norm / 4)
    assert got.shape() == [] and abs(got.data()[0] - norm) <= 2.0 ** -22 * norm
    np.testing.assert_allclose(grad(a), before / 4, rtol=2.0 ** -21)
    assert np.array_equal(grad(b), other)
    y = tensor(f(rng, 50))
    y.mul(y).sum().backward()  # 2 y, not stored
    assert abs(K.grad_norm([y]).data()[0] - 2 * np.linalg.norm(y.data().astype(np.float64))) <= 1e-5
    K.clip_grad_norm([y, b], 0.5)
    both = np.concatenate([grad(y), grad(b)]).astype(np.float64)
    assert abs(np.linalg.norm(both) - 0.5) <= 1e-6
    assert K.grad_norm([]).data()[0] == 0


def test_training_and_serving_together():
    """norm -> product -> norm, gate, residual -> norm -> product -> loss; backward, the clipped step; then the trained
    weights in 8 bits.  The same steps in 64 bits beside it."""
    rng = np.random.default_rng(8)
    rows, cols, classes, lr, max_norm = 64, 96, 32, 0.05, 0.75
    a = {"w0": f(rng, cols, mean=1.0, std=0.1), "m1": f(rng, cols, cols, std=0.1), "gate": f(rng, cols, mean=1.0, std=0.1),
         "w1": f(rng, cols, mean=1.0, std=0.1), "w2": f(rng, cols, mean=1.0, std=0.1), "m2": f(rng, cols, classes, std=0.1)}
    x = f(rng, rows, cols)
    t = {k: tensor(v) for k, v in a.items()}
    exact = {k: v.astype(np.float64) for k, v in a.items()}
    xt, x64 = tensor(x), x.astype(np.float64)
    for step in range(3):
        for v in t.values():
            v.zero_grad()
        n0 = K.Norm(t["w0"]).forward(xt)
        r, n = K.BlockNorm(K.Norm(t["w1"]), K.Norm(t["w2"]), 0.5).forward(xt, n0.matmul(t["m1"]), t["gate"])
        out = n.matmul(t["m2"])
        out.mul(out).sum().backward()
        norm = K.sgd_step_clipped(list(t.values()), lr, max_norm)
        # 64 bits
        e = exact
        n0_ = block_ref.norm(x64, e["w0"], None, 1e-6, False)
        h_ = n0_ @ e["m1"]
        gate = e["gate"][None]
        r_, n_ = block_ref.forward(x64, h_, gate, e["w1"], None, e["w2"], None, 0.5, 1e-6, False)
        out_ = n_ @ e["m2"]
        g_out = 2 * out_
        b = block_ref.backward(r_, h_, gate, e["w1"], None, e["w2"], 0.5, 1e-6, False, None, g_out @ e["m2"].T)
        grads = {"m2": n_.T @ g_out, "w2": b["dpre_w"], "w1": b["dpost_w"], "gate": b["dgate"][0], "m1": n0_.T @ b["dh"]}
        grads["w0"] = block_ref.norm_vjp(x64, e["w0"], b["dh"] @ e["m1"].T, 1e-6, False)[1]
        total = np.sqrt(sum(np.square(v).sum() for v in grads.values()))
        assert abs(norm.data()[0] - total) <= TOL * total, step
        for k, v in grads.items():
            assert rel_l2(grad(t[k]), v) <= 3 * TOL, (step, k)
            e[k] = e[k] - lr * min(1.0, max_norm / total) * v
            assert rel_l2(t[k].data(), e[k]) <= TOL, (step, k)
    served = K.Int8Linear(t["m2"])
    assert (served.in_features(), served.out_features()) == (cols, classes)
    for m in (1, rows):
        rows_n = n.data().reshape(rows, cols)[:m]
        y = served.forward(tensor(rows_n))
        xq, xs = block_ref.quantize(rows_n)
        wq, ws = block_ref.quantize(t["m2"].data().reshape(cols, classes).T)
        assert rel_l2(y.data(), block_ref.int8_product(xq, xs, wq, ws, None)) <= 4 * 2.0 ** -24
        assert y.op() == K.Op.Leaf and y.parents() == []
    before = t["m2"].data().copy()
    t["m2"].sgd_step(1.0)  # what was quantised stays
    assert not np.array_equal(before, t["m2"].data())
    assert np.array_equal(served.forward(tensor(rows_n)).data(), y.data())
