"""Gradients of gradients through layer_norm, embedding_lookup and distillation_loss, on the numpy stand-in
backend: an outer gradients() has to see everything that an inner one computes from its leaves.

The truth is float64: the first gradients from their formulas, differentiated by the complex step (exact to
rounding, no difference is taken).  The stand-in rounds every result to float32; a nested gradient here is a
chain of at most 64 of them with terms of up to 8 times the result's largest value: 64 * 8 * 2^-24 of that."""
import numpy as np
import pytest

from test_token_ops_host import TokenBackend
from tfjs_core_b200 import ops
from tfjs_core_b200.engine import ENGINE

TOL = 64 * 8 * 2.0 ** -24


class EmptyRowsBackend(TokenBackend):
    """Like the kernels, exactly 0 in the rows whose list is empty, whatever their logits hold."""

    def _there(self, logits, indices):
        i = self._i(indices)
        return ((i >= 0) & (i < logits.shape[-1])).any(-1)

    def distillationLoss(self, logits, teacherLogits, teacherIndices, temperature=1.0, withStats=True):
        loss, stats = super().distillationLoss(logits, teacherLogits, teacherIndices, temperature, withStats)
        return self._make(np.where(self._there(logits, teacherIndices), self._v(loss), 0)), stats

    def distillationLossBackprop(self, dloss, logits, teacherLogits, teacherIndices, stats, temperature=1.0):
        dz = super().distillationLossBackprop(dloss, logits, teacherLogits, teacherIndices, stats, temperature)
        return self._make(np.where(self._there(logits, teacherIndices)[..., None], self._v(dz), 0))


@pytest.fixture()
def host():
    prev = ENGINE.backendName
    bk = EmptyRowsBackend()
    ENGINE.registerBackend("numpy-token-nested-test", lambda: bk, 1000)
    assert ENGINE.setBackend("numpy-token-nested-test")
    yield bk
    ENGINE.removeBackend("numpy-token-nested-test")
    if prev:
        ENGINE.setBackend(prev)


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


def _check(f, gradients, arrays, rng, tol=TOL):
    weights = [rng.normal(0, 1, a.shape).astype(np.float32) for a in arrays]
    want = _second(gradients, [a.astype(np.float64) for a in arrays], [w.astype(np.float64) for w in weights])
    tensors = [ops.tensor(a) for a in arrays]
    before = ENGINE.numTensors
    got = ENGINE.tidy(lambda: ops.grads(_nested(f, weights))(tensors))
    assert ENGINE.numTensors == before + len(got)   # the inner tape leaves nothing behind
    for g, w in zip(got, want):
        assert g.shape == list(w.shape)
        np.testing.assert_allclose(g.dataSync().reshape(w.shape), w, rtol=0, atol=tol * np.abs(w).max())


def test_embedding_lookup(host):
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


def test_embedding_lookup_three_times(host):
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
def test_layer_norm(host, weights):
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


def test_layer_norm_over_several_axes(host):
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


def test_layer_norm_three_times(host):
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


def _distillation_gradient(z, u, idx, dloss, t):
    """dloss t (q - p) of rows [rows, classes]; complex z allowed."""
    e = np.exp(z / t - (z.real / t).max(-1, keepdims=True))
    q = e / e.sum(-1, keepdims=True)
    ok = (idx >= 0) & (idx < z.shape[-1])
    w = np.where(ok, np.exp(u.astype(np.float64) / t), 0)
    some = ok.any(-1, keepdims=True)
    w = w / np.where(some, w.sum(-1, keepdims=True), 1)
    p = np.zeros(z.shape)
    for r, k in zip(*np.nonzero(ok)):
        p[r, idx[r, k]] += w[r, k]
    return np.where(some, dloss[:, None] * t * (q - p), 0)


def _distillation_case(rng):
    z = rng.normal(0, 1, (4, 6)).astype(np.float32)
    idx = np.stack([rng.permutation(6)[:3] for _ in range(4)]).astype(np.int32)
    idx[1] = -1                      # no teacher
    idx[2, 1] = idx[2, 0]            # a class named twice
    idx[3, 2] = 6                    # a shorter list
    return z, rng.normal(0, 1, (4, 3)).astype(np.float32), idx


@pytest.mark.parametrize("t", [1.0, 2.5])
def test_distillation_loss(host, t):
    rng = np.random.default_rng(3)
    z, u, idx = _distillation_case(rng)
    tu, ti = ops.tensor(u), ops.tensor(idx, dtype="int32")

    # f = sum(c(z) loss(z)) + sum(z^2), c = (sum z)^2 of the row: the inner dloss depends on the logits too
    def f(v):
        c = ops.square(ops.sum(v, [1]))
        return ops.add(ops.sum(ops.mul(c, ops.distillation_loss(v, tu, ti, t))), ops.sum(ops.square(v)))

    def gradients(v):
        s = v.sum(-1)
        log_q = v / t - np.log(np.exp(v / t).sum(-1, keepdims=True))
        ok = (idx >= 0) & (idx < 6)
        w = np.where(ok, np.exp(u.astype(np.float64) / t), 0)
        p = w / np.maximum(w.sum(-1, keepdims=True), 1e-300)
        gap = np.log(np.where(p > 0, p, 1)) - np.take_along_axis(log_q, np.where(ok, idx, 0), -1)
        loss = t * t * (p * gap).sum(-1)
        return [_distillation_gradient(v, u, idx, s * s, t) + (2 * s * loss)[:, None] + 2 * v]
    _check(f, gradients, [z], rng)


def test_distillation_loss_leaves_out_rows_without_a_teacher(host):
    """What such a row's logits hold does not matter to a nested gradient either."""
    rng = np.random.default_rng(4)
    z, u, idx = _distillation_case(rng)
    w = rng.normal(0, 1, z.shape).astype(np.float32)
    tu, ti, tw = ops.tensor(u), ops.tensor(idx, dtype="int32"), ops.tensor(w)
    outer = lambda v: ops.sum(ops.mul(ops.grad(lambda s: ops.sum(ops.distillation_loss(s, tu, ti)))(v), tw))  # noqa: E731
    want = ops.grad(outer)(ops.tensor(z)).dataSync().reshape(z.shape)
    z[1, 2] = np.nan
    got = ops.grad(outer)(ops.tensor(z)).dataSync().reshape(z.shape)
    assert not got[1].any() and np.array_equal(got, want)


def test_distillation_loss_three_times(host):
    """Two classes with logits (t, 0) and the teacher on the second: loss = log(1 + e^t); its derivatives
    along (1, 0) are s, s (1 - s) and s (1 - s) (1 - 2 s), s = 1 / (1 + e^-t).  The teacher of the second row
    is equal over both classes, like its student: q - p is 0 there, its derivative is not."""
    u, ti = ops.tensor(np.zeros((2, 2), np.float32)), ops.tensor(np.array([[1, -1], [0, 1]]), dtype="int32")
    e = ops.tensor(np.array([[1.0, 0.0], [1.0, 0.0]], np.float32))
    t = np.array([0.4, 0.0])
    x = ops.tensor(np.stack([t, 0 * t], -1).astype(np.float32))
    along = lambda h: (lambda v: ops.sum(ops.mul(ops.grad(lambda s: ops.sum(h(s)))(v), e), [1]))  # noqa: E731
    f = lambda v: ops.distillation_loss(v, u, ti)  # noqa: E731
    s = 1 / (1 + np.exp(-t))
    first = s - np.array([0, 0.5])
    for want in (first, s * (1 - s), s * (1 - s) * (1 - 2 * s)):
        f = along(f)
        np.testing.assert_allclose(f(x).dataSync(), want, rtol=0, atol=TOL)


def test_single_rows_without_a_batch_axis(host):
    rng = np.random.default_rng(6)
    z, u = rng.normal(0, 1, 5).astype(np.float32), rng.normal(0, 1, 2).astype(np.float32)
    idx = np.array([4, 1], np.int32)
    tu, ti = ops.tensor(u), ops.tensor(idx, dtype="int32")
    f = lambda v: ops.distillation_loss(ops.layer_norm(v, epsilon=0.1), tu, ti, 2.0)  # noqa: E731

    def gradients(v):
        n, _ = _normalised(v[None], 0.1)
        dz = _distillation_gradient(n, u[None], idx[None], np.ones(1), 2.0)
        return [_layer_norm_gradients(dz, v[None], np.ones(5), 0.1)[0][0]]
    _check(f, gradients, [z], rng)
    table = rng.normal(0, 1, (3, 2)).astype(np.float32)
    at = ops.scalar(2, "int32")
    got = ops.grad(lambda t: ops.sum(ops.grad(lambda s: ops.sum(ops.square(ops.embedding_lookup(s, at))))(t)))(ops.tensor(table))
    np.testing.assert_array_equal(got.dataSync().reshape(3, 2), [[0, 0], [0, 0], [2, 2]])
