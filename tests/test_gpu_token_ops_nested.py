"""Gradients of gradients through layer_norm, embedding_lookup and distillation_loss on the device, against
float64.  The kernels take exp and log as good to 2^-21 where the host stand-in rounds to 2^-24: eight times
its tolerance."""
import numpy as np
import pytest

import test_token_ops_nested as nested
from gpu_util import tf  # noqa: F401
from tfjs_core_b200 import ops

pytestmark = pytest.mark.gpu
TOL = 8 * nested.TOL


def test_model_differentiated_twice(tf):
    """table -> lookup -> layerNorm -> logits -> distillationLoss, with respect to table, gamma and beta."""
    rng = np.random.default_rng(7)
    tokens, vocab, width, t = 9, 5, 6, 2.0
    idx = np.array([0, 1, 1, 4, -1, 2, 2, 2, 7], np.int32)
    classes = np.stack([rng.permutation(width)[:3] for _ in range(tokens)]).astype(np.int32)
    classes[2, 1:], classes[4], classes[5, 1] = -1, -1, classes[5, 0]
    u = rng.normal(0, 1, (tokens, 3)).astype(np.float32)
    table = rng.normal(0, 1, (vocab, width)).astype(np.float32)
    gamma, beta = rng.normal(1, 0.3, width).astype(np.float32), rng.normal(0, 0.3, width).astype(np.float32)
    ti, tu, tc = ops.tensor(idx, dtype="int32"), ops.tensor(u), ops.tensor(classes, dtype="int32")

    def f(p, g, b):
        e = ops.embedding_lookup(p, ti, 1.5)
        loss = ops.distillation_loss(ops.layer_norm(e, g, b, epsilon=0.1), tu, tc, t)
        return ops.add(ops.sum(loss), ops.sum(ops.square(p)))

    def gradients(p, g, b):
        ok = (idx >= 0) & (idx < vocab)
        e = np.where(ok[:, None], 1.5 * p[np.where(ok, idx, 0)], 0)
        z = nested._normalised(e, 0.1)[0] * g + b
        dz = nested._distillation_gradient(z, u, classes, np.ones(tokens), t)
        de, dg, db = nested._layer_norm_gradients(dz, e, g, 0.1)
        dp = 2 * p
        np.add.at(dp, idx[ok], 1.5 * de[ok])
        return [dp, dg, db]
    nested._check(f, gradients, [table, gamma, beta], rng, TOL)


def test_half_storage_mode_keeps_nested_gradients_in_float32(tf):
    bk = tf.ENGINE.backend
    rng = np.random.default_rng(8)
    table = rng.normal(0, 1, (5, 4)).astype(np.float32)
    ti = ops.tensor(np.array([0, 3, 3], np.int32), dtype="int32")
    w = rng.normal(0, 1, (5, 4)).astype(np.float32)
    # d/dt of sum(w grad(sum(e s))) with s = sum(t): the inner gradient is s times counts + sum(e); the derivative of
    # sum(w s counts) is sum(w counts) everywhere and that of sum(w) sum(e) is sum(w) counts
    counts = np.array([1, 0, 0, 2, 0.0])[:, None]
    want = (w * counts).sum(dtype=np.float64) + w.sum(dtype=np.float64) * counts * np.ones((5, 4))
    bk.setActivationStorage("float16")
    try:
        inner = lambda t: ops.mul(ops.sum(ops.embedding_lookup(t, ti)), ops.sum(t))  # noqa: E731
        g = ops.grad(lambda t: ops.sum(ops.mul(ops.grad(inner)(t), ops.tensor(w))))(ops.tensor(table))
    finally:
        bk.setActivationStorage("float32")
    assert bk._rec(g.dataId)["dtype"] == "float32"
    # float32 sums of at most 20 terms, 80 roundings in all; a rounding to half on the way would be 2^-12
    np.testing.assert_allclose(g.dataSync().reshape(5, 4), want, rtol=0, atol=80 * 2.0 ** -24 * np.abs(w).sum())


def test_rows_without_a_teacher_and_special_logits(tf):
    rng = np.random.default_rng(9)
    z, u, idx = nested._distillation_case(rng)
    w = rng.normal(0, 1, z.shape).astype(np.float32)
    tu, ti, tw = ops.tensor(u), ops.tensor(idx, dtype="int32"), ops.tensor(w)
    outer = lambda v: ops.sum(ops.mul(ops.grad(lambda s: ops.sum(ops.distillation_loss(s, tu, ti)))(v), tw))  # noqa: E731
    want = ops.grad(outer)(ops.tensor(z)).dataSync().reshape(z.shape)
    z[1, 2] = np.nan
    got = ops.grad(outer)(ops.tensor(z)).dataSync().reshape(z.shape)
    assert not got[1].any() and np.array_equal(got, want) and want[0].any()
