"""Nested gradients through ops that save their own result (exp, softmax): the saved clone has to stay
connected to the op's inputs, at every order.  Expected values are closed forms; tolerances count float32
roundings (at most 32, of terms up to 4 times the result)."""
import numpy as np
import pytest

from numpy_backend import NumpyBackend
from tfjs_core_b200 import ops
from tfjs_core_b200.engine import ENGINE

RTOL = 32 * 4 * 2.0 ** -24


class SoftmaxBackend(NumpyBackend):
    def softmax(self, x):
        v = self._v(x).astype(np.float64)
        e = np.exp(v - v.max(-1, keepdims=True))
        return self._make(e / e.sum(-1, keepdims=True))


@pytest.fixture()
def host():
    prev = ENGINE.backendName
    bk = SoftmaxBackend()
    ENGINE.registerBackend("numpy-nested-test", lambda: bk, 1000)
    assert ENGINE.setBackend("numpy-nested-test")
    yield bk
    ENGINE.removeBackend("numpy-nested-test")
    if prev:
        ENGINE.setBackend(prev)


def _derivatives(f, x, n):
    out = []
    for _ in range(n + 1):
        out.append(float(f(ops.scalar(x)).dataSync()[0]))
        f = ops.grad(f)
    return out


def test_exp(host):
    x = 0.7
    want = [np.exp(x) * (x + k) for k in range(4)]
    np.testing.assert_allclose(_derivatives(lambda t: ops.mul(ops.exp(t), t), x, 3), want, rtol=RTOL)
    want = np.array([1, 2 * x, 4 * x * x + 2, 8 * x ** 3 + 12 * x]) * np.exp(x * x)
    np.testing.assert_allclose(_derivatives(lambda t: ops.exp(ops.square(t)), x, 3), want, rtol=RTOL)


def test_softmax_hessian(host):
    z = np.array([0.3, -0.4, 1.1], np.float32)
    v, w = np.array([1.0, -2.0, 0.5]), np.array([0.2, 1.5, -1.0])
    tv, tw = ops.tensor(v), ops.tensor(w)
    f = lambda t: ops.sum(ops.mul(ops.fused_softmax(t), tv))  # noqa: E731
    before = ENGINE.numTensors
    g = ops.grad(lambda t: ENGINE.tidy(lambda: ops.sum(ops.mul(ops.grad(f)(t), tw))))(ops.tensor(z))
    q = np.exp(z.astype(np.float64))
    q /= q.sum()
    # y . J(q) w, J = diag(q) - q q^T, differentiated once more
    a, b, ab = v - q @ v, w - q @ w, q @ (v * w) - (q @ v) * (q @ w)
    want = q * (a * b - ab)
    np.testing.assert_allclose(g.dataSync(), want, rtol=0, atol=RTOL * np.abs(want).max())
    g.dispose()
    assert ENGINE.numTensors == before + 1   # the argument of the call


def test_first_gradients_and_saved_tensors_are_as_before(host):
    x = ops.tensor(np.array([[0.5, -1.0], [2.0, 3.0]], np.float32))
    before, buffers = ENGINE.numTensors, len(host.data)
    value, (g,) = ops.value_and_grads(lambda t: ops.sum(ops.mul(ops.exp(t), t)))([x])
    v = np.array([0.5, -1.0, 2.0, 3.0])
    np.testing.assert_allclose(g.dataSync(), np.exp(v) * (v + 1), rtol=RTOL)
    value.dispose()
    g.dispose()
    assert ENGINE.numTensors == before and len(host.data) == buffers
