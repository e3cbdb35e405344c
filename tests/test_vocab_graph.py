"""Embedding, DistillLoss and adjust_logits on the graph, alone and in the steps that a language model takes with them."""
import numpy as np
import pytest

import block_ref
import katsu_b200 as K
import vocab_ref as ref
from parity_util import rel_l2

# f32 chains over rows of up to 96 values; products in 3xTF32 mode hold 1e-5 by their documents
TOL = 1e-5


def f(rng, *shape, mean=0.0, std=1.0):
    return (mean + std * rng.standard_normal(shape)).astype(np.float32)


def tensor(a):
    return K.Tensor(a, list(a.shape))


def grad(t):
    g = t.grad()
    return None if g is None else g.reshape(t.shape())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(), (1,), (5, 7), (2, 3, 4), (0,), (300,)])
def test_embedding(shape):
    rng = np.random.default_rng(1)
    table, tokens = f(rng, 20, 12), rng.integers(-1, 20, shape)
    c = f(rng, *shape, 12)
    t = tensor(table)
    y = K.Embedding(t, 3.0).forward(tokens)
    assert y.shape() == [*shape, 12] and y.op() == K.Op("Embed", scale=3.0) and y.parents()[0].id() == t.id()
    assert np.array_equal(y.data().reshape(c.shape), ref.embed(table, tokens.reshape(-1), 3.0).astype(np.float32).reshape(c.shape))
    y.mul(tensor(c)).sum().backward()
    want, off = ref.embed_grad(tokens.reshape(-1), c.reshape(-1, 12), 3.0, 20)
    ref.assert_near(grad(t), want, off)


@pytest.mark.gpu
def test_a_table_with_two_uses():
    """Two lookups and a product of one table: three contributions to one gradient, and a table that is no leaf."""
    rng = np.random.default_rng(2)
    a, b = f(rng, 9, 8), f(rng, 9, 8)
    first, second = rng.integers(0, 9, 30), rng.integers(0, 9, 400)
    ta, tb = tensor(a), tensor(b)
    table = ta.add(tb)
    layer = K.Embedding(table, 0.5)
    c, d, e = f(rng, 30, 8), f(rng, 400, 8), f(rng, 8, 5)
    loss = layer.forward(first).mul(tensor(c)).sum().add(layer.forward(second).mul(tensor(d)).sum()).add(table.matmul(tensor(e)).sum())
    loss.backward()
    want = sum(ref.embed_grad(t, g, 0.5, 9)[0] for t, g in ((first, c), (second, d))) + e.astype(np.float64).sum(1)
    assert rel_l2(grad(table), want) <= TOL and rel_l2(grad(ta), want) <= TOL and rel_l2(grad(tb), want) <= TOL


@pytest.mark.gpu
@pytest.mark.parametrize("shape,top,T,soft,hard", [((6,), 5, 2.0, 0.5, 0.5), ((2, 3), 4, 1.0, 1.0, 0.0), ((), 3, 1.5, 1.0, 0.2), ((8,), 0, 1.0, 0.0, 1.0)])
@pytest.mark.parametrize("weighted", [False, True])
def test_distill_loss(shape, top, T, soft, hard, weighted):
    rng = np.random.default_rng(3)
    rows, vocab = int(np.prod(shape)), 50
    z, teacher, index, labels = f(rng, rows, vocab), f(rng, rows, top), rng.integers(-1, vocab, (rows, top)), rng.integers(-1, vocab, rows)
    weight, g = f(rng, rows), f(rng, rows)
    t = K.Tensor(z, [*shape, vocab])
    layer = K.DistillLoss(T, soft, hard)
    loss = layer.forward(t, K.Tensor(teacher, [*shape, top]) if top else None, index if top else None, labels, tensor(weight) if weighted else None)
    assert loss.shape() == list(shape) and loss.op().kind == "Distill" and loss.op().temperature == np.float32(T)
    loss.mul(K.Tensor(g, list(shape))).sum().backward()
    want, off, dz, doff = ref.distill(z, teacher, index, labels, weight if weighted else None, T, soft, hard, g)
    ref.assert_near(loss.data(), want, off)
    ref.assert_near(t.grad(), dz, doff)


@pytest.mark.gpu
def test_logits_with_two_uses():
    rng = np.random.default_rng(4)
    z, labels, c = f(rng, 7, 33), rng.integers(0, 33, 7), f(rng, 7, 33)
    t = tensor(z)
    layer = K.DistillLoss(1.0, 0.0, 1.0)
    layer.forward(t, labels=labels).sum().add(t.mul(tensor(c)).sum()).add(layer.forward(t, labels=labels[::-1].copy()).sum()).backward()
    one = [ref.distill(z, np.zeros((7, 0)), np.zeros((7, 0), int), v, None, 1.0, 0.0, 1.0)[2] for v in (labels, labels[::-1])]
    assert rel_l2(grad(t), one[0] + one[1] + c) <= TOL


@pytest.mark.gpu
def test_adjusted_logits_and_a_served_head():
    """A decoding step of a model served in 8 bits: lookup from the head's weights, norm, head, adjusted logits."""
    rng = np.random.default_rng(5)
    k, vocab, rows = 48, 100, 4
    w, norm_w = f(rng, k, vocab), f(rng, k, mean=1.0)
    head = K.Int8Linear(tensor(w))
    tokens = rng.integers(0, vocab, rows)
    x = head.embed(tokens, 2.0)
    q, s = block_ref.quantize(w.T)
    want = (q[tokens].astype(np.float32) * s[tokens][:, None]) * np.float32(2)
    assert x.shape() == [rows, k] and x.op() == K.Op.Leaf and np.array_equal(x.data().reshape(rows, k), want)
    logits = head.forward(K.Norm(tensor(norm_w)).forward(x))
    history, lengths, prompts = rng.integers(-1, vocab, (rows, 20)), np.array([20, 0, 7, 13]), np.array([5, 0, 9, 0])
    allowed = rng.random((rows, vocab)) < 0.5
    bias_tokens, bias = rng.integers(-1, vocab, (rows, 3)), f(rng, rows, 3)
    got = K.adjust_logits(logits, history, lengths, prompts, 1.2, 0.3, [0.1, 0.2, 0.3, 0.4], bias_tokens, bias, allowed)
    full = lambda v: np.full(rows, v, np.float32)  # noqa: E731
    z = logits.data().reshape(rows, vocab)
    want, off = ref.adjust(z, history, prompts, lengths, full(1.2), full(0.3), np.float32([0.1, 0.2, 0.3, 0.4]), bias_tokens, bias, allowed)
    assert got.shape() == [rows, vocab] and got.op() == K.Op.Leaf
    ref.assert_near(got.data(), want, off)
    alone = K.adjust_logits(K.Tensor(z[0], [vocab]), history[:1], lengths[:1], prompts[:1], 1.2, 0.3, [0.1], bias_tokens[:1], bias[:1], allowed[0])
    assert alone.shape() == [vocab] and np.array_equal(alone.data(), got.data().reshape(rows, vocab)[0])
    assert np.array_equal(K.adjust_logits(logits).data().reshape(rows, vocab), z)


@pytest.mark.gpu
@pytest.mark.parametrize("T,hard", [(1.0, 0.0), (2.0, 0.5)])
def test_a_training_step_of_a_small_model(T, hard):
    """Tokens in, a teacher's top logits out: lookup, norm, product, residual and norm, head, loss, and a clipped step of everything.
    Every gradient against the formulas in 64 bits."""
    rng = np.random.default_rng(6)
    rows, vocab, cols, top, scale, eps = 40, 60, 32, 6, 4.0, 1e-6
    a = {"table": f(rng, vocab, cols, std=0.3), "norm": f(rng, cols, mean=1.0, std=0.2), "w": f(rng, cols, cols, std=cols ** -0.5),
         "last": f(rng, cols, mean=1.0, std=0.2), "head": f(rng, cols, vocab, std=cols ** -0.5)}
    tokens, labels = ref.zipf(rng, vocab, rows), rng.integers(-1, vocab, rows)
    teacher, index = f(rng, rows, top, std=2.0), np.stack([rng.permutation(vocab)[:top] for _ in range(rows)])
    weight = np.full(rows, 1.0 / rows, np.float32)
    weight[::9] = 0
    t = {k: tensor(v) for k, v in a.items()}
    x = K.Embedding(t["table"], scale).forward(tokens)
    h = K.Norm(t["norm"], eps=eps).forward(x).matmul(t["w"])
    r, n = K.BlockNorm(None, K.Norm(t["last"], eps=eps)).forward(x, h)
    logits = n.matmul(t["head"])
    loss = K.DistillLoss(T, 1 - hard, hard).forward(logits, tensor(teacher), index, labels, tensor(weight))
    loss.sum().backward()
    # the same in 64 bits
    d = {k: v.astype(np.float64) for k, v in a.items()}
    x64 = ref.embed(a["table"], tokens, scale)
    n1 = block_ref.norm(x64, d["norm"], None, eps, False)
    r64, n64 = block_ref.forward(x64, n1 @ d["w"], None, None, None, d["last"], None, 1.0, eps, False)
    want, off, dz, _ = ref.distill(n64 @ d["head"], teacher, index, labels, weight, T, 1 - hard, hard)
    assert rel_l2(loss.data(), want) <= TOL
    grads = {"head": n64.T @ dz}
    dr, grads["last"], _ = block_ref.norm_vjp(r64, d["last"], dz @ d["head"].T, eps, False)
    grads["w"] = n1.T @ dr
    dx, grads["norm"], _ = block_ref.norm_vjp(x64, d["norm"], dr @ d["w"].T, eps, False)
    grads["table"] = np.zeros((vocab, cols))
    np.add.at(grads["table"], tokens, scale * (dr + dx))
    for name, g in grads.items():
        assert rel_l2(grad(t[name]), g) <= 2 * TOL, name  # two products one behind the other
    norm = float(np.sqrt(sum(np.square(g).sum() for g in grads.values())))
    got = K.sgd_step_clipped(list(t.values()), 0.1, norm / 2)
    assert abs(float(got.data()[0]) - norm) <= 2 * TOL * norm
    for name, g in grads.items():
        assert rel_l2(t[name].data(), a[name] - 0.1 * 0.5 * g) <= 2 * TOL, name


@pytest.mark.gpu
def test_operands_that_are_refused():
    t = K.Tensor.zeros([6, 4])
    with pytest.raises(K.RankMismatch):
        K.Embedding(K.Tensor.zeros([4]))
    with pytest.raises(K.InvalidOperand, match="token 6 of a vocabulary of 6"):
        K.Embedding(t).forward([1, 6])
    with pytest.raises(K.InvalidOperand, match="whole numbers"):
        K.Embedding(t).forward([0.5])
    with pytest.raises(K.InvalidOperand):
        K.Embedding(t).forward([2 ** 40])
    with pytest.raises(K.InvalidOperand, match="token 4"):
        K.Int8Linear(t).embed([4])
    for T, soft, hard in ((0.0, 1, 0), (-1.0, 1, 0), (float("nan"), 1, 0), (float("inf"), 1, 0), (1.0, float("inf"), 0), (1.0, 1, float("nan"))):
        with pytest.raises(K.InvalidOperand):
            K.DistillLoss(T, soft, hard)
    layer = K.DistillLoss()
    with pytest.raises(K.InvalidOperand, match="last axis"):
        layer.forward(K.Tensor.zeros([]))
    with pytest.raises(K.InvalidOperand, match="last axis"):
        layer.forward(K.Tensor.zeros([3, 0]))
    with pytest.raises(K.InvalidOperand, match="axes"):
        layer.forward(t, K.Tensor.zeros([5, 2]), np.zeros((5, 2), int))
    with pytest.raises(K.InvalidOperand, match="axes"):
        layer.forward(t, K.Tensor.zeros([6]), np.zeros(6, int))
    with pytest.raises(K.InvalidOperand, match="at most"):
        layer.forward(t, K.Tensor.zeros([6, 1025]), np.zeros((6, 1025), int))
    with pytest.raises(K.DataLength):
        layer.forward(t, K.Tensor.zeros([6, 2]), np.zeros((6, 1), int))
    with pytest.raises(K.DataLength):
        layer.forward(t, labels=[1])
    with pytest.raises(K.DataLength):
        layer.forward(t, labels=[1] * 6, weight=K.Tensor.zeros([5]))
    with pytest.raises(K.InvalidOperand, match="label 4"):
        layer.forward(t, labels=[4] * 6)
    with pytest.raises(K.InvalidOperand, match="index 9"):
        layer.forward(t, K.Tensor.zeros([6, 1]), [[9]] * 6)
    for bad in ({"history": [[1, 2]] * 5}, {"repetition": [1.0, 2.0]}, {"lengths": [1]}, {"bias": [[1.0]] * 6}, {"bias": [1.0], "bias_tokens": [1]},
                {"allowed": np.ones((6, 3), bool)}, {"history": [[4]] * 6}, {"bias": np.zeros((6, 1025)), "bias_tokens": np.zeros((6, 1025), int)}):
        with pytest.raises((K.InvalidOperand, K.DataLength)):
            K.adjust_logits(t, **bad)
    with pytest.raises(K.RankMismatch):
        K.adjust_logits(K.Tensor.zeros([2, 3, 4]))


@pytest.mark.gpu
def test_nothing_to_do():
    empty = K.adjust_logits(K.Tensor.zeros([0, 5]))
    assert empty.shape() == [0, 5]
    loss = K.DistillLoss(1.0, 0.0, 1.0).forward(K.Tensor.zeros([0, 5]), labels=[])
    assert loss.shape() == [0]
    t = K.Tensor.zeros([0, 4])
    y = K.Embedding(t).forward([-1, -5])
    assert y.shape() == [2, 4] and not y.data().any()
    y.sum().backward()
    assert t.grad() is not None and t.grad().size == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [[0, 5], [2, 0], [0, 0], [0]])
def test_masks_of_nothing(shape):
    out = K.adjust_logits(K.Tensor.zeros(shape), allowed=np.zeros(shape, bool), repetition=1.5)
    assert out.shape() == shape and out.data().size == 0
    with pytest.raises(K.InvalidOperand):
        K.adjust_logits(K.Tensor.zeros(shape), allowed=np.zeros([*shape, 1], bool))


@pytest.mark.parametrize("shape", [[], [2, 3, 4]])
def test_masks_of_other_ranks(shape):
    with pytest.raises(K.RankMismatch):
        K.adjust_logits(K.Tensor.zeros(shape), allowed=np.ones(shape, bool))
