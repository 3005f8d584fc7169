"""Gradients of gradients through layer_norm, embedding_lookup and distillation_loss, on the numpy stand-in
backend: an outer gradients() has to see everything that an inner one computes from its leaves.

The truth is float64: the first gradients from their formulas, differentiated by the complex step (exact to
rounding, no difference is taken).  The stand-in rounds every result to float32; a nested gradient here is a
chain of at most 64 of them with terms of up to 8 times the result's largest value: 64 * 8 * 2^-24 of that."""
import numpy as np
import pytest

from test_token_ops_host import host  # noqa: F401  (the fixture)
from tfjs_core_b200 import ops
from tfjs_core_b200.engine import ENGINE

TOL = 64 * 8 * 2.0 ** -24


def _directional(gradients, arrays, i, at):
    """d gradients(arrays) / d arrays[i][at] by the complex step."""
    moved = [a.astype(np.complex128) for a in arrays]
    moved[i][at] += 1e-30j
    return [g.imag / 1e-30 for g in gradients(*moved)]


def _second(gradients, arrays, weights):
    """The gradients of sum_j sum(weights[j] * gradients(arrays)[j]) with respect to each array."""
    out = []
    for i, a in enumerate(arrays):
        g = np.zeros(a.shape)
        for at in np.ndindex(*a.shape):
            g[at] = sum((w * d).sum() for w, d in zip(weights, _directional(gradients, arrays, i, at)))
        out.append(g)
    return out


def _nested(f, weights):
    """sum_j sum(weights[j] * grad_j f), as a function of f's arguments."""
    def outer(*xs):
        total = None
        for g, w in zip(ops.grads(f)(list(xs)), weights):
            term = ops.sum(ops.mul(g, ops.tensor(w)))
            total = term if total is None else ops.add(total, term)
        return total
    return outer


def _check(f, gradients, arrays, rng):
    weights = [rng.normal(0, 1, a.shape).astype(np.float32) for a in arrays]
    want = _second(gradients, [a.astype(np.float64) for a in arrays], [w.astype(np.float64) for w in weights])
    tensors = [ops.tensor(a) for a in arrays]
    before = ENGINE.numTensors
    got = ENGINE.tidy(lambda: ops.grads(_nested(f, weights))(tensors))
    assert ENGINE.numTensors == before + len(got)   # the inner tape leaves nothing behind
    for g, w in zip(got, want):
        assert g.shape == list(w.shape)
        np.testing.assert_allclose(g.dataSync().reshape(w.shape), w, rtol=0, atol=TOL * np.abs(w).max())


def test_embedding_lookup(host):  # noqa: F811
    rng = np.random.default_rng(0)
    table = rng.normal(0, 1, (5, 3)).astype(np.float32)
    idx = np.array([[1, 1], [4, -1], [7, 0]])      # a row named twice, two indices outside the table
    ti = ops.tensor(idx, dtype="int32")
    v = rng.normal(0, 1, (3, 2, 3)).astype(np.float32)

    # f = sum(v e^3) + sum(t^2), e = 1.5 t[i]: the second path keeps the outer tape connected by itself
    def f(t):
        e = ops.embedding_lookup(t, ti, 1.5)
        return ops.add(ops.sum(ops.mul(ops.tensor(v), ops.mul(e, ops.square(e)))), ops.sum(ops.square(t)))

    def gradients(t):
        ok = (idx >= 0) & (idx < 5)
        e = np.where(ok[..., None], 1.5 * t[np.where(ok, idx, 0)], 0)
        out = 2 * t
        np.add.at(out, idx[ok], (1.5 * 3 * v * e * e)[ok])
        return [out]
    _check(f, gradients, [table], rng)


def test_embedding_lookup_three_times(host):  # noqa: F811
    """d^3/dt^3 of sum(e^4) along ones, e = 2 t[i]: 24 * 2^4 t for each place that names the row."""
    t = np.array([[1.0], [-2.0], [0.5]], np.float32)
    ti = ops.tensor(np.array([0, 2, 2, 3]), dtype="int32")
    f = lambda x: ops.sum(ops.square(ops.square(ops.embedding_lookup(x, ti, 2.0))))  # noqa: E731
    g = ops.grad(ops.grad(ops.grad(f)))(ops.tensor(t))
    np.testing.assert_allclose(g.dataSync(), [384.0, 0.0, 384.0], rtol=TOL)


def _normalised(x, epsilon):
    c = x - x.mean(-1, keepdims=True)
    r = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + epsilon)
    return c * r, r


def _layer_norm_gradients(dy, x, gamma, epsilon):
    n, r = _normalised(x, epsilon)
    a = dy * gamma
    dx = r * (a - a.mean(-1, keepdims=True) - n * (a * n).mean(-1, keepdims=True))
    return dx, (dy * n).sum(0), dy.sum(0)


@pytest.mark.parametrize("weights", [True, False])
def test_layer_norm(host, weights):  # noqa: F811
    rng = np.random.default_rng(1)
    x = rng.normal(0.5, 1, (3, 5)).astype(np.float32)
    g, b = rng.normal(1, 0.3, 5).astype(np.float32), rng.normal(0, 0.3, 5).astype(np.float32)
    v = rng.normal(0, 1, (3, 5)).astype(np.float32)

    # f = sum(v y^2) + sum(x^2), y = layer_norm(x, g, b): dy depends on y, and so on all three leaves
    def f(p, q=None, s=None):
        y = ops.layer_norm(p, q, s, epsilon=0.1)
        return ops.add(ops.sum(ops.mul(ops.tensor(v), ops.square(y))), ops.sum(ops.square(p)))

    def gradients(p, q=np.ones(5), s=np.zeros(5)):
        dx, dg, db = _layer_norm_gradients(2 * v * (_normalised(p, 0.1)[0] * q + s), p, q, 0.1)
        return [dx + 2 * p, dg, db][:3 if weights else 1]
    _check(f, gradients, [x, g, b] if weights else [x], rng)


def test_layer_norm_over_several_axes(host):  # noqa: F811
    rng = np.random.default_rng(2)
    x = rng.normal(0, 1, (2, 3, 2)).astype(np.float32)
    g, v = rng.normal(1, 0.3, (3, 2)).astype(np.float32), rng.normal(0, 1, (2, 3, 2)).astype(np.float32)

    def f(p, q):
        return ops.sum(ops.mul(ops.tensor(v), ops.square(ops.layer_norm(p, q, axis=[1, 2], epsilon=0.1))))

    def gradients(p, q):
        x2, g1 = p.reshape(2, 6), q.reshape(6)
        dx, dg, _ = _layer_norm_gradients(2 * v.reshape(2, 6) * _normalised(x2, 0.1)[0] * g1, x2, g1, 0.1)
        return [dx.reshape(p.shape), dg.reshape(q.shape)]
    _check(f, gradients, [x, g], rng)


def test_layer_norm_three_times(host):  # noqa: F811
    """Row [t, 0, -t], epsilon 1: y_0 = t / sqrt(2 t^2 / 3 + 1) along (1, 0, -1); the third derivative of y_0 in
    t is the sum of the third partial derivatives along it, taken here as nested gradients along that direction."""
    t, e = 0.7, np.array([1.0, 0.0, -1.0], np.float32)
    along = lambda h: (lambda x: ops.sum(ops.mul(ops.grad(h)(x), ops.tensor(e))))  # noqa: E731
    f = lambda x: ops.sum(ops.mul(ops.layer_norm(x, epsilon=1.0), ops.tensor(np.array([1.0, 0, 0], np.float32))))  # noqa: E731
    got = float(along(along(along(f)))(ops.tensor(t * e)).dataSync()[0])
    # d^3/dt^3 of t (1 + c t^2)^-1/2, c = 2/3: (12 c^2 t^2 - 3 c) (1 + c t^2)^-7/2
    c = 2 / 3
    want = (12 * c * c * t * t - 3 * c) * (1 + c * t * t) ** -3.5
    assert abs(got - want) <= 4 * TOL * 3 * c   # the two terms of the numerator cancel in part
