"""grad_norm, clip_grad_norm and sgd_step_clipped take any iterable of tensors, one that makes them on the way included."""
import weakref

import numpy as np
import pytest

import katsu_b200 as K


class Passing:
    """Stands for a tensor that only the iterable holds."""

    def __init__(self, handle):
        self._h = handle


class Library:
    """Looks, while it is called, whether the tensors behind the handles still live."""

    def __init__(self, made):
        self.made, self.alive = made, []

    def kh_grad_norm(self, handles, count, *rest):
        self.alive = [ref() is not None for ref in self.made]
        self.seen = list(handles[:count])
        return 1

    kh_clip_grad_norm = kh_sgd_step_clipped = kh_grad_norm


@pytest.mark.parametrize("call", [lambda t: K.grad_norm(t), lambda t: K.clip_grad_norm(t, 1.0), lambda t: K.sgd_step_clipped(t, 0.1, 1.0)],
                         ids=["norm", "clip", "step"])
def test_tensors_live_while_the_library_is_called(call, monkeypatch):
    made = []

    def passing():
        for handle in (16, 32, 48):
            t = Passing(handle)
            made.append(weakref.ref(t))
            yield t

    library = Library(made)
    monkeypatch.setattr(K, "_load", lambda: library)

    class Reached(Exception):
        pass

    def check(rc):
        raise Reached()

    monkeypatch.setattr(K, "_check", check)
    with pytest.raises(Reached):
        call(passing())
    assert library.seen == [16, 32, 48] and library.alive == [True] * 3


@pytest.mark.gpu
def test_parents_of_a_node():
    a, b = (K.Tensor(np.arange(1, 4, dtype=np.float32), [3]) for _ in range(2))
    y = a.add(b)
    y.sum().backward()
    assert abs(K.grad_norm(t for t in y.parents()).data()[0] - 6 ** 0.5) <= 2.0 ** -22 * 6 ** 0.5
    K.sgd_step_clipped((t for t in y.parents()), 1.0, 100.0)
    assert np.array_equal(a.data(), [0, 1, 2]) and np.array_equal(b.data(), [0, 1, 2])
