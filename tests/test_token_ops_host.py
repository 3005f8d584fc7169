"""layer_norm, embedding_lookup and distillation_loss in the op layer, on a numpy stand-in backend: the
tape's nodes and their gradients against differences, several normalised axes, lifetimes, refusals."""
import numpy as np
import pytest

from numpy_backend import NumpyBackend
from tfjs_core_b200 import ops
from tfjs_core_b200.engine import ENGINE


class TokenBackend(NumpyBackend):
    """The six kernels in float64 numpy, written from their formulas."""

    def _i(self, t):
        return self.data[t.dataId].reshape(t.shape).astype(np.int64)

    def layerNorm(self, x, gamma, beta, epsilon, withStats=False, outputStorage=None):
        v = self._v(x).astype(np.float64)
        m = v.mean(-1, keepdims=True)
        r = 1 / np.sqrt(((v - m) ** 2).mean(-1, keepdims=True) + epsilon)
        y = (v - m) * r * (1 if gamma is None else self._v(gamma)) + (0 if beta is None else self._v(beta))
        return self._make(y), self._make(np.concatenate([m, r], -1)) if withStats else None

    def layerNormBackprop(self, dy, x, gamma, stats):
        d, v, s = (self._v(t).astype(np.float64) for t in (dy, x, stats))
        n = (v - s[..., :1]) * s[..., 1:]
        a = d * (1 if gamma is None else self._v(gamma))
        dx = s[..., 1:] * (a - a.mean(-1, keepdims=True) - n * (a * n).mean(-1, keepdims=True))
        axes = tuple(range(d.ndim - 1))
        return self._make(dx), self._make((d * n).sum(axes)), self._make(d.sum(axes))

    def embeddingLookup(self, table, indices, scale=1.0, outputStorage=None):
        w, i = self._v(table), self._i(indices)
        ok = (i >= 0) & (i < w.shape[0])
        return self._make(np.where(ok[..., None], w[np.where(ok, i, 0)] * scale, 0))

    def embeddingLookupBackprop(self, dy, indices, vocab, scale=1.0):
        d, i = self._v(dy), self._i(indices)
        ok = (i >= 0) & (i < vocab)
        out = np.zeros((vocab, d.shape[-1]))
        np.add.at(out, i[ok], d[ok] * float(scale))
        return self._make(out)

    def _distillation(self, logits, u, indices, t):
        z, u, i = self._v(logits).astype(np.float64) / t, self._v(u).astype(np.float64) / t, self._i(indices)
        log_q = z - z.max(-1, keepdims=True)
        log_q = log_q - np.log(np.exp(log_q).sum(-1, keepdims=True))
        ok = (i >= 0) & (i < z.shape[-1])
        e = np.where(ok, np.exp(np.where(ok, u, 0)), 0)
        p = e / np.maximum(e.sum(-1, keepdims=True), 1e-300)
        return log_q, np.where(ok, i, 0), p

    def distillationLoss(self, logits, teacherLogits, teacherIndices, temperature=1.0, withStats=True):
        log_q, i, p = self._distillation(logits, teacherLogits, teacherIndices, temperature)
        gap = np.log(np.where(p > 0, p, 1)) - np.take_along_axis(log_q, i, -1)
        loss = temperature ** 2 * (p * gap).sum(-1)
        return self._make(loss), self._make(np.zeros(loss.shape + (4,))) if withStats else None

    def distillationLossBackprop(self, dloss, logits, teacherLogits, teacherIndices, stats, temperature=1.0):
        log_q, i, p = self._distillation(logits, teacherLogits, teacherIndices, temperature)
        d = np.exp(log_q) * (p.sum(-1, keepdims=True) > 0)
        flat, rows = d.reshape(-1, d.shape[-1]), np.arange(d[..., 0].size)
        for k in range(p.shape[-1]):
            flat[rows, i.reshape(-1, p.shape[-1])[:, k]] -= p.reshape(-1, p.shape[-1])[:, k]
        return self._make(d * self._v(dloss)[..., None] * temperature)


@pytest.fixture()
def host():
    prev = ENGINE.backendName
    bk = TokenBackend()
    ENGINE.registerBackend("numpy-token-test", lambda: bk, 1000)
    assert ENGINE.setBackend("numpy-token-test")
    yield bk
    ENGINE.removeBackend("numpy-token-test")
    if prev:
        ENGINE.setBackend(prev)


def _differences(f, arrays, i, h=1e-2):
    """Central differences of sum f(arrays) with respect to arrays[i] (the backend rounds to float32)."""
    g = np.zeros(arrays[i].shape)
    for at in np.ndindex(*g.shape):
        side = []
        for s in (h, -h):
            a = [v.copy() for v in arrays]
            a[i][at] += s
            side.append(float(ENGINE.tidy(lambda: f(*[ops.tensor(v) for v in a])).dataSync().astype(np.float64).sum()))
        g[at] = (side[0] - side[1]) / (2 * h)
    return g


def _check(f, arrays, tol):
    before = ENGINE.numTensors
    tensors = [ops.tensor(v) for v in arrays]
    value, grads = ops.value_and_grads(f)(tensors)
    for i, g in enumerate(grads):
        assert g.shape == list(arrays[i].shape)
        np.testing.assert_allclose(g.dataSync().reshape(arrays[i].shape), _differences(f, arrays, i), atol=tol)
    for t in tensors + grads + [value]:
        t.dispose()
    return before


def test_layer_norm_gradients_over_one_and_several_axes(host):
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (2, 3, 4)).astype(np.float32)
    w = rng.normal(0, 1, (2, 3, 4)).astype(np.float32)
    for axis, shape in ((-1, (4,)), ([1, 2], (3, 4)), ([0, 1, 2], (2, 3, 4)), ([2, 1], (3, 4))):
        g, b = rng.normal(1, 0.2, shape).astype(np.float32), rng.normal(0, 0.2, shape).astype(np.float32)
        tw = ops.tensor(w)
        # differences of step h = 1e-2 on float32 values of order 1: h^2 times third derivatives and 1e-7 / h
        _check(lambda p, q, r: ops.mul(ops.layer_norm(p, q, r, axis=axis, epsilon=0.1), tw), [x, g, b], 5e-3)
        y = ops.layer_norm(ops.tensor(x), ops.tensor(g), ops.tensor(b), axis=axis)
        assert y.shape == [2, 3, 4]
    plain = ops.layer_norm(ops.tensor(x)).dataSync().reshape(x.shape)
    np.testing.assert_allclose(plain, (x - x.mean(-1, keepdims=True)) / np.sqrt(x.var(-1, keepdims=True) + 1e-5), atol=1e-5)


def test_embedding_and_distillation_gradients(host):
    rng = np.random.default_rng(1)
    table = rng.normal(0, 1, (5, 3)).astype(np.float32)
    idx = ops.tensor(np.array([[1, 1], [4, -1], [7, 0]]), dtype="int32")
    _check(lambda t: ops.square(ops.embedding_lookup(t, idx, 1.5)), [table], 5e-3)
    z = rng.normal(0, 1, (2, 3, 6)).astype(np.float32)
    ti = np.stack([[rng.permutation(6)[:2] for _ in range(3)] for _ in range(2)]).astype(np.int32)
    ti[0, 1], ti[1, 0, 1] = -1, ti[1, 0, 0]      # an empty list, and a class named twice
    u, i = ops.tensor(rng.normal(0, 1, (2, 3, 2))), ops.tensor(ti, dtype="int32")
    for t in (1.0, 2.0):
        _check(lambda v: ops.distillation_loss(v, u, i, t), [z], 5e-3)
    assert ops.distillation_loss(ops.tensor(z), u, i).shape == [2, 3]


def test_nothing_leaks_and_nothing_is_saved_without_a_tape(host):
    x, g = ops.tensor(np.ones((2, 4), np.float32)), ops.tensor(np.ones(4, np.float32))
    i = ops.tensor(np.array([0, 1]), dtype="int32")
    u, c = ops.tensor(np.ones((2, 1), np.float32)), ops.tensor(np.zeros((2, 1)), dtype="int32")
    before, buffers = ENGINE.numTensors, len(host.data)
    for f, xs in ((lambda p, q: ops.layer_norm(p, q, q), [x, g]), (lambda p: ops.embedding_lookup(p, i), [x]),
                  (lambda p: ops.distillation_loss(p, u, c), [x])):
        f(*xs).dispose()
        assert ENGINE.numTensors == before and len(host.data) == buffers
        value, grads = ops.value_and_grads(f)(xs)
        for t in grads + [value]:
            t.dispose()
        assert ENGINE.numTensors == before and len(host.data) == buffers


def test_the_teacher_is_a_constant(host):
    z, u = ops.tensor(np.ones((2, 4), np.float32)), ops.tensor(np.ones((2, 1), np.float32))
    c = ops.tensor(np.zeros((2, 1)), dtype="int32")
    with pytest.raises(ValueError, match="Cannot compute gradient"):
        ops.grad(lambda t: ops.distillation_loss(z, t, c))(u)


def test_refusals(host):
    x = ops.tensor(np.ones((2, 3, 4), np.float32))
    four = ops.tensor(np.ones(4, np.float32))
    with pytest.raises(ValueError, match="inner-most"):
        ops.layer_norm(x, axis=1)
    with pytest.raises(ValueError, match="inner-most"):
        ops.layer_norm(x, axis=[])
    with pytest.raises(ValueError, match="inner-most"):
        ops.layer_norm(ops.scalar(1.0))
    with pytest.raises(ValueError, match="gamma must have shape"):
        ops.layer_norm(x, four, axis=[1, 2])
    with pytest.raises(ValueError, match="beta must have shape"):
        ops.layer_norm(x, None, ops.tensor(np.ones(3, np.float32)))
    with pytest.raises(ValueError, match="epsilon"):
        ops.layer_norm(x, epsilon=-1.0)
    i = ops.tensor(np.zeros(3), dtype="int32")
    with pytest.raises(ValueError, match="rank 2"):
        ops.embedding_lookup(x, i)
    with pytest.raises(ValueError, match="int32"):
        ops.embedding_lookup(ops.tensor(np.ones((4, 2), np.float32)), ops.tensor(np.zeros(3)))
    z = ops.tensor(np.ones((3, 5), np.float32))
    u, c = ops.tensor(np.ones((3, 2), np.float32)), ops.tensor(np.zeros((3, 2)), dtype="int32")
    with pytest.raises(ValueError, match="must be"):
        ops.distillation_loss(z, ops.tensor(np.ones((2, 2), np.float32)), c)
    with pytest.raises(ValueError, match="must be"):
        ops.distillation_loss(z, u, ops.tensor(np.zeros((3, 1)), dtype="int32"))
    with pytest.raises(ValueError, match="int32"):
        ops.distillation_loss(z, u, ops.tensor(np.zeros((3, 2))))
    with pytest.raises(ValueError, match="temperature"):
        ops.distillation_loss(z, u, c, 0.0)
