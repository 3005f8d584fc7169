"""layerNorm, embeddingLookup and distillationLoss with their gradients against plain float64 numpy.

Tolerances are bounds, not fits.  u = 2^-24 is half a float32 step.  A float32 sum of n terms whose
longest chain of additions is D is off by at most D u sum|terms| (first order); the kernels' chains
stay below CHAIN.  A value stored as half is off by 2^-11 of itself more (2^-25 below the normals).
exp and log are taken as good to 2^-21 relative and absolute."""
import ctypes as C

import numpy as np
import pytest

from gpu_util import tf  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CHAIN = 256
FN = 2.0 ** -21


def _rng(*seed):
    return np.random.Generator(np.random.PCG64(list(seed)))


def _stored(bk, a, storage):
    return bk.registerStored(list(a.shape), storage, a)


def _as_stored(a, storage):
    a = np.asarray(a, np.float32)
    return a.astype(np.float16).astype(np.float32) if storage == "float16" else a


def _half_step(v, storage):
    return np.abs(v) * 2.0 ** -11 + 2.0 ** -25 if storage == "float16" else 0.0


def _within(got, want, tol):
    got = np.asarray(got, np.float64).reshape(want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    same = np.isnan(want) | fine
    assert np.array_equal(got[~same], want[~same])
    over = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)) - np.broadcast_to(tol, want.shape), 0)
    at = np.unravel_index(np.argmax(over), over.shape) if over.size else ()
    assert not over.size or over[at] <= 0, (at, got[at], want[at], np.broadcast_to(tol, want.shape)[at])


# ---- layer normalisation ---------------------------------------------------------------------------
EPS = 1e-5


def _ln_reference(x, g, b):
    x = x.astype(np.float64)
    m = x.mean(-1, keepdims=True)
    r = 1 / np.sqrt(((x - m) ** 2).mean(-1, keepdims=True) + EPS)
    n = (x - m) * r
    y = n * g.astype(np.float64) + b.astype(np.float64)
    # |mean off| <= CHAIN u max|x|, rstd off by half as much relatively plus its own rounding
    off = np.abs(g) * (r * CHAIN * U * np.abs(x).max(-1, keepdims=True) + (CHAIN / 2 + 8) * U * np.abs(n)) + 2 * U * (np.abs(y) + np.abs(b))
    return y, off, m[..., 0], r[..., 0]


LN_SHAPES = [(1, 1), (3, 1), (1, 1024), (5, 3), (7, 8), (130, 32), (33, 48), (64, 64), (19, 100), (301, 128), (9, 255),
             (77, 256), (150, 300), (40, 512), (29, 768), (301, 1000), (6, 1001), (10, 1024), (13, 1028), (9, 1536),
             (5, 2048), (200, 2050), (3, 4096), (4, 4104), (301, 5000), (2, 8192), (3, 8200), (2, 10001), (2, 16384),
             (1, 16392), (3, 25088), (2, 50177), (1, 100352), (2, 131072), (1, 262147), (160, 9000), (1, 600000), (150, 66), (50, 114), (400, 130), (90, 515), (70, 1023), (70, 1030), (40, 2046),
             (40, 2047), (30, 3001), (30, 4098), (20, 6143), (20, 8191), (12, 16383), (6, 16386), (150, 16400), (150, 20003),
             (40, 33000), (30, 50002), (160, 8200)]


@pytest.mark.parametrize("rows,width", LN_SHAPES)
@pytest.mark.parametrize("sx,sy", [("float32", "float32"), ("float16", "float16"), ("float16", "float32"), ("float32", "float16")])
def test_layer_norm(tf, rows, width, sx, sy):
    bk = tf.ENGINE.backend
    rng = _rng(rows, width)
    x = _as_stored(rng.normal(0.5, 2, (rows, width)), sx)
    g, b = rng.normal(1, 0.3, width).astype(np.float32), rng.normal(0, 0.3, width).astype(np.float32)
    y, stats = bk.layerNorm(_stored(bk, x, sx), tf.ops.tensor(g), tf.ops.tensor(b), EPS, True, sy)
    want, off, m, r = _ln_reference(x, g, b)
    assert bk._rec(y.dataId)["dtype"] == sy
    _within(y.dataSync(), want, off + _half_step(want, sy))
    s = stats.dataSync().reshape(rows, 2)
    _within(s[:, 0], m, CHAIN * U * np.abs(x).max(-1))
    # d(var) / (var + eps) <= CHAIN u, halved by the root; plus the mean's own error, squared, is below that
    _within(s[:, 1], r, (CHAIN / 2 + 8) * U * r)


def test_layer_norm_without_weights_and_statistics(tf):
    bk = tf.ENGINE.backend
    for rows, width in [(5, 24), (3, 515), (2, 3000), (2, 40000)]:
        x = _rng(width).normal(0, 1, (rows, width)).astype(np.float32)
        one, zero = np.ones(width, np.float32), np.zeros(width, np.float32)
        g = _rng(1).normal(1, 0.2, width).astype(np.float32)
        tx = tf.ops.tensor(x)
        for gamma, beta in [(None, None), (g, None), (None, g)]:
            want, off, _, _ = _ln_reference(x, one if gamma is None else gamma, zero if beta is None else beta)
            y, stats = bk.layerNorm(tx, None if gamma is None else tf.ops.tensor(gamma),
                                    None if beta is None else tf.ops.tensor(beta), EPS)
            assert stats is None
            _within(y.dataSync(), want, off)


def test_layer_norm_of_constant_rows_large_means_and_special_values(tf):
    bk = tf.ENGINE.backend
    for width in (16, 1000, 4096, 40000):
        x = np.zeros((6, width), np.float32)
        x[0] = 3.0                                            # variance 0
        x[1] = 1e4 + _rng(width).normal(0, 1, width)          # mean far above the spread
        x[2] = _rng(width + 1).normal(0, 1e-20, width)        # squares underflow: rstd = eps^-1/2
        x[3] = _rng(2).normal(0, 1, width)
        x[3, width // 2] = np.nan
        x[4] = x[3, 0]
        x[4, 0] = np.inf
        x[5] = _rng(3).normal(0, 1, width)
        one, zero = np.ones(width, np.float32), np.zeros(width, np.float32)
        y, stats = bk.layerNorm(tf.ops.tensor(x), None, None, EPS, True)
        got, s = y.dataSync().reshape(x.shape), stats.dataSync().reshape(6, 2)
        good = [0, 1, 2, 5]
        want, off, m, r = _ln_reference(x[good], one, zero)
        _within(got[good], want, off)
        assert abs(s[0, 0] - 3.0) == 0 and np.all(got[0] == 0)
        assert np.isnan(got[3]).all() and np.isnan(got[4]).all() and np.isnan(s[3:5, 1]).all()


def _ln_backward_reference(dy, x, g, stats):
    dy, x, g, stats = (v.astype(np.float64) for v in (dy, x, g, stats))
    m, r = stats[:, :1], stats[:, 1:]
    n, a = (x - m) * r, dy * g
    n_off = 2 * U * r * (np.abs(x) + np.abs(m)) + 2 * U * np.abs(n)
    ma, man = a.mean(-1, keepdims=True), (a * n).mean(-1, keepdims=True)
    ma_off = CHAIN * U * np.abs(a).mean(-1, keepdims=True)
    man_off = CHAIN * U * np.abs(a * n).mean(-1, keepdims=True) + (np.abs(a) * n_off).mean(-1, keepdims=True)
    dx = r * (a - ma - n * man)
    dx_off = r * (2 * U * np.abs(a) + ma_off + np.abs(n) * man_off + n_off * np.abs(man) + 4 * U * (np.abs(a) + np.abs(ma) + np.abs(n * man)))
    dg, db = (dy * n).sum(0), dy.sum(0)
    dg_off = CHAIN * U * np.abs(dy * n).sum(0) + (np.abs(dy) * n_off).sum(0)
    return (dx, dx_off), (dg, dg_off), (db, CHAIN * U * np.abs(dy).sum(0) + U * np.abs(db))


@pytest.mark.parametrize("rows,width", LN_SHAPES + [(3001, 64), (5000, 8), (2049, 1024), (1500, 1030)])
@pytest.mark.parametrize("sd,sx", [("float32", "float32"), ("float32", "float16"), ("float16", "float16"), ("float16", "float32")])
def test_layer_norm_backprop(tf, rows, width, sd, sx):
    bk = tf.ENGINE.backend
    rng = _rng(rows, width, 5)
    x, dy = _as_stored(rng.normal(0.5, 2, (rows, width)), sx), _as_stored(rng.normal(0, 1, (rows, width)), sd)
    g = rng.normal(1, 0.3, width).astype(np.float32)
    stats = np.stack([x.mean(-1), 1 / np.sqrt(x.var(-1) + EPS)], -1).astype(np.float32)
    tensors = _stored(bk, dy, sd), _stored(bk, x, sx), tf.ops.tensor(g), tf.ops.tensor(stats)
    out = bk.layerNormBackprop(*tensors)
    for got, (want, off) in zip(out, _ln_backward_reference(dy, x, g, stats)):
        _within(got.dataSync(), want, off)
    again = bk.layerNormBackprop(*tensors)
    for a, b in zip(out, again):   # the same bits on every run
        assert np.array_equal(a.dataSync(), b.dataSync())


def test_layer_norm_backprop_without_gamma_and_with_outputs_left_out(tf):
    bk = tf.ENGINE.backend
    lib, ctx = bk._lib, bk._ctx
    for rows, width in [(37, 96), (300, 1024), (5, 3001), (2, 20000)]:
        rng = _rng(rows)
        x, dy = rng.normal(0, 1, (2, rows, width)).astype(np.float32)
        stats = np.stack([x.mean(-1), 1 / np.sqrt(x.var(-1) + EPS)], -1).astype(np.float32)
        td, tx, ts = (tf.ops.tensor(v) for v in (dy, x, stats))
        want = _ln_backward_reference(dy, x, np.ones(width, np.float32), stats)
        for got, (w, off) in zip(bk.layerNormBackprop(td, tx, None, ts), want):
            _within(got.dataSync(), w, off)
        sizes = [[rows, width], [width], [width]]
        for keep in range(3):
            outs = [tf.ops.tensor(np.full(s, 7, np.float32)) for s in sizes]
            ids = [bk._oid(t) if i == keep else 0 for i, t in enumerate(outs)]
            assert lib.tfjs_cuda_layer_norm_backprop(ctx, bk._oid(td), bk._oid(tx), 0, bk._oid(ts), *ids, rows, width) == 0
            for i, (t, (w, off)) in enumerate(zip(outs, want)):
                if i == keep:
                    _within(t.dataSync(), w, off)
                else:
                    assert np.all(t.dataSync() == 7)


# ---- embedding lookup ------------------------------------------------------------------------------
TABLES = [(1, 1), (7, 3), (50, 4), (33, 8), (100, 63), (1000, 64), (257, 100), (1000, 130), (300, 256), (64, 1000), (40, 2049)]


def _tokens(rng, count, vocab):
    i = np.minimum(np.exp(rng.uniform(0, np.log(vocab + 1), count)).astype(np.int64) - 1, vocab - 1).astype(np.int32)
    for at, v in ((3, -1), (5, vocab), (9, -2 ** 31), (11, 2 ** 31 - 1), (12, vocab - 1), (13, 0)):
        if at < count:
            i[at] = v
    return i


@pytest.mark.parametrize("vocab,width", TABLES)
@pytest.mark.parametrize("count", [1, 37, 1025])
@pytest.mark.parametrize("st,so", [("float32", "float32"), ("float16", "float16"), ("uint8", "float32"), ("uint8", "float16"),
                                   ("float16", "float32"), ("float32", "float16")])
def test_embedding_lookup(tf, vocab, width, count, st, so):
    bk = tf.ENGINE.backend
    rng = _rng(vocab, width, count)
    idx = _tokens(rng, count, vocab)
    scale = np.float32(width ** 0.5)
    if st == "uint8":
        q = rng.integers(0, 256, (vocab, width)).astype(np.uint8)
        table = bk.registerQuantized([vocab, width], q, 0.0173, -2.2)
        values = (q.astype(np.float64) * 0.0173 + -2.2).astype(np.float32)
    else:
        values = _as_stored(rng.normal(0, 1, (vocab, width)), st)
        table = _stored(bk, values, st)
    out = bk.embeddingLookup(table, tf.ops.tensor(idx, dtype="int32"), float(scale), so)
    ok = (idx >= 0) & (idx < vocab)
    want = np.where(ok[:, None], values[np.where(ok, idx, 0)] * scale, np.float32(0))
    assert out.shape == [count, width] and bk._rec(out.dataId)["dtype"] == so
    # one float32 product, one rounding to the storage: bit for bit
    assert np.array_equal(out.dataSync().reshape(want.shape), _as_stored(want, so))


@pytest.mark.parametrize("vocab,width", TABLES + [(100003, 24), (300000, 5)])
@pytest.mark.parametrize("count", [1, 31, 64, 1025, 9000])
@pytest.mark.parametrize("sd", ["float32", "float16"])
def test_embedding_lookup_backprop(tf, vocab, width, count, sd):
    bk = tf.ENGINE.backend
    rng = _rng(vocab, width, count, 7)
    idx = _tokens(rng, count, vocab)
    dy = _as_stored(rng.normal(0, 1, (count, width)), sd)
    scale = np.float32(1.7)
    args = _stored(bk, dy, sd), tf.ops.tensor(idx, dtype="int32"), vocab, float(scale)
    out = bk.embeddingLookupBackprop(*args)
    ok = (idx >= 0) & (idx < vocab)
    want, total = np.zeros((2, vocab, width))
    named = np.zeros((vocab, 1))
    np.add.at(want, idx[ok], dy[ok].astype(np.float64) * scale)
    np.add.at(total, idx[ok], np.abs(dy[ok]).astype(np.float64) * scale)
    np.add.at(named, idx[ok], 1)
    _within(out.dataSync(), want, (named + 2) * U * total)   # at worst one chain over the row's tokens
    assert np.array_equal(out.dataSync(), bk.embeddingLookupBackprop(*args).dataSync())


@pytest.mark.parametrize("count,vocab,width", [(70001, 300, 8), (70001, 1, 4), (66000, 150000, 4), (65536, 70000, 4),
                                               (65537, 70000, 3), (20000, 2, 260), (40000, 5, 33), (300000, 1 << 20, 1)])
def test_embedding_lookup_backprop_of_many_tokens(tf, count, vocab, width):
    bk = tf.ENGINE.backend
    rng = _rng(count, vocab, width, 9)
    idx = _tokens(rng, count, vocab)
    idx[-count // 10:] = -1
    dy = rng.normal(0, 1, (count, width)).astype(np.float32)
    out = bk.embeddingLookupBackprop(tf.ops.tensor(dy), tf.ops.tensor(idx, dtype="int32"), vocab)
    ok = (idx >= 0) & (idx < vocab)
    want, total = np.zeros((2, vocab, width))
    np.add.at(want, idx[ok], dy[ok].astype(np.float64))
    np.add.at(total, idx[ok], np.abs(dy[ok]).astype(np.float64))
    named = np.bincount(idx[ok], minlength=vocab)[:, None]
    _within(out.dataSync(), want, (named + 2) * U * total)


@pytest.mark.parametrize("count", [1, 16, 17, 1000, 8192, 40000, 65536, 66000])
@pytest.mark.parametrize("token", [-1, 0, 4, 5])
def test_embedding_gradient_of_one_token_throughout(tf, count, token):
    bk = tf.ENGINE.backend
    dy = _rng(count).normal(0, 1, (count, 20)).astype(np.float32)
    idx = np.full(count, token, np.int32)
    got = bk.embeddingLookupBackprop(tf.ops.tensor(dy), tf.ops.tensor(idx, dtype="int32"), 5, 0.5).dataSync().reshape(5, 20)
    want, off = np.zeros((2, 5, 20))
    if 0 <= token < 5:
        want[token] = dy.astype(np.float64).sum(0) * 0.5
        # chains: 32 tokens a share, an eighth of the shares a warp, 8 warps
        off[token] = (32 + count / 256 + 16) * U * np.abs(dy).sum(0) * 0.5 + U * np.abs(want[token])
    _within(got, want, off)


def test_embedding_gradient_keeps_special_values_in_their_rows(tf):
    bk = tf.ENGINE.backend
    idx = np.array([2, 0, 2, -1, 0, 5], np.int32)
    dy = np.ones((6, 8), np.float32)
    dy[0, 1], dy[1, 2], dy[3], dy[5, 0] = np.nan, np.inf, np.nan, -np.inf
    got = bk.embeddingLookupBackprop(tf.ops.tensor(dy), tf.ops.tensor(idx, dtype="int32"), 6, 2.0).dataSync().reshape(6, 8)
    want = np.zeros((6, 8), np.float32)
    want[0], want[2], want[5] = 4, 4, 2
    want[2, 1], want[0, 2], want[5, 0] = np.nan, np.inf, -np.inf
    assert np.array_equal(got, want, equal_nan=True)


# ---- distillation loss -----------------------------------------------------------------------------
def _distillation_reference(z, u, idx, dloss, t):
    z, u, dloss = z.astype(np.float64) / t, u.astype(np.float64) / t, dloss.astype(np.float64)
    rows, classes = z.shape
    with np.errstate(divide="ignore", invalid="ignore"):
        m = z.max(-1, keepdims=True)
        lse = m + np.log(np.exp(z - m).sum(-1, keepdims=True))
        log_q = z - lse
        ok = (idx >= 0) & (idx < classes) & (u != -np.inf)
        at = np.where(ok, idx, 0)
        some = ok.any(-1)
        v = np.where(ok, u, -np.inf)
        vm = np.where(some, v.max(-1, initial=-np.inf), 0)[:, None]
        e = np.exp(v - vm)
        total = np.where(some, e.sum(-1), 1)[:, None]
        p, log_p = e / total, v - vm - np.log(total)
        gap = np.where(p > 0, log_p - np.take_along_axis(log_q, at, -1), 0)
        loss = t * t * np.where(p > 0, p * gap, 0).sum(-1)
        q = np.exp(log_q)
        target = np.zeros_like(z)
        for k in range(idx.shape[1]):
            target[np.arange(rows), at[:, k]] += np.where(ok[:, k], p[:, k], 0)
        dz = (dloss * t)[:, None] * (q - target)
        # the logarithm of a sum is off by the sum's relative error plus the rounding of the largest z
        big = np.where(np.isfinite(z), np.abs(z), 0).max(-1, initial=0)
        ubig = np.where(ok & np.isfinite(u), np.abs(u), 0).max(-1, initial=0)
        es, et = (8 * big + CHAIN) * U + 2 * FN, (8 * ubig + CHAIN) * U + 2 * FN
        loss_off = t * t * ((es + et) + (et + CHAIN * U) * np.where(p > 0, p * np.abs(gap), 0).sum(-1))
        dz_off = np.abs(dloss * t)[:, None] * ((es[:, None] + 8 * U) * q + (et[:, None] + (8 + idx.shape[1]) * U) * target) + 2.0 ** -126
    for v in (loss, loss_off, dz, dz_off):   # exactly 0 where the teacher has nothing to say
        v[~some] = 0
    return loss, loss_off, dz, dz_off, lse[:, 0]


def _teacher(rng, rows, classes, top):
    idx = np.stack([rng.permutation(classes)[:top] if classes >= top else rng.integers(0, classes, top) for _ in range(rows)])
    return idx.astype(np.int32), -np.sort(-rng.normal(0, 3, (rows, top)), -1)


def _check_distillation(tf, z, u, idx, t, sz, su, dloss=None):
    bk = tf.ENGINE.backend
    rows, classes = z.shape
    z, u = _as_stored(z, sz), _as_stored(u, su)
    if dloss is None:
        dloss = _rng(rows).uniform(0.2, 1, rows).astype(np.float32)
    tz, tu, ti, td = _stored(bk, z, sz), _stored(bk, u, su), tf.ops.tensor(idx, dtype="int32"), tf.ops.tensor(dloss)
    loss, stats = bk.distillationLoss(tz, tu, ti, t)
    dz = bk.distillationLossBackprop(td, tz, tu, ti, stats, t)
    want, off, dwant, doff, lse = _distillation_reference(z, u, idx, dloss, t)
    _within(loss.dataSync(), want, off)
    _within(dz.dataSync(), dwant, doff)
    assert dz.shape == [rows, classes]
    loss2, none = bk.distillationLoss(tz, tu, ti, t, False)
    assert none is None and np.array_equal(loss.dataSync(), loss2.dataSync(), equal_nan=True)
    assert np.array_equal(dz.dataSync(), bk.distillationLossBackprop(td, tz, tu, ti, stats, t).dataSync(), equal_nan=True)
    return loss.dataSync(), dz.dataSync().reshape(rows, classes)


@pytest.mark.parametrize("rows,classes,top", [(1, 1, 1), (3, 2, 1), (5, 7, 7), (64, 10, 3), (33, 100, 5), (128, 1000, 5),
                                              (7, 1001, 64), (2, 4099, 32), (300, 515, 9), (5, 32000, 64), (2, 32001, 128),
                                              (1, 131101, 1), (2, 150000, 1024), (700, 2048, 17), (9, 12345, 0),
                                              (1300, 1025, 128), (1300, 5001, 5), (1250, 8192, 3), (1200, 8193, 2), (40, 3000, 129)])
@pytest.mark.parametrize("sz,su", [("float32", "float32"), ("float16", "float16"), ("float16", "float32"), ("float32", "float16")])
def test_distillation_loss(tf, rows, classes, top, sz, su):
    rng = _rng(rows, classes, top)
    idx, u = _teacher(rng, rows, classes, top)
    _check_distillation(tf, rng.normal(0, 2, (rows, classes)), u, idx, [1.0, 2.0, 0.7][top % 3], sz, su)


@pytest.mark.parametrize("classes", [9, 1000, 40000])
def test_distillation_of_short_empty_and_repeated_lists(tf, classes):
    rng = _rng(classes)
    rows, top = 10, 6
    z = rng.normal(0, 2, (rows, classes))
    idx, u = _teacher(rng, rows, classes, top)
    idx[0, 4:] = -1                      # a short list
    idx[1] = -1                          # none
    u[2] = -np.inf                       # listed, but masked out
    idx[3] = idx[3, 0]                   # one class six times
    idx[4, 3], idx[4, 5] = idx[4, 0], idx[4, 1]
    idx[5, 2], u[5, 2] = -1, np.nan      # what a masked entry holds does not matter
    idx[6, 1], u[6, 1] = classes, np.inf
    idx[7, 0], u[7, 0] = -2 ** 31, np.nan
    u[8, 2:] = np.finfo(np.float32).min  # masked by the type's lowest value
    z[9] = 3.5                           # no class preferred
    loss, dz = _check_distillation(tf, z, u, idx, 2.0, "float32", "float32")
    assert loss[1] == 0 and loss[2] == 0 and not dz[1].any() and not dz[2].any()


def test_distillation_with_masked_classes_and_special_logits(tf):
    for classes in (12, 1000, 33000):
        rng = _rng(classes, 3)
        z = rng.normal(0, 2, (6, classes))
        idx, u = _teacher(rng, 6, classes, 4)
        z[0, [c for c in range(classes // 2) if c not in idx[0]]] = -np.inf   # masked classes: q = 0
        z[1, [c for c in range(classes // 2) if c not in idx[1]]] = np.finfo(np.float32).min
        z[2, idx[2, 0]] = -np.inf                                             # the teacher wants a masked class
        z[3, 5] = np.nan
        z[4] = -np.inf                                                        # nothing left to the student
        idx[5] = -1
        z[5, 2] = np.nan                                                      # but nobody asks
        loss, dz = _check_distillation(tf, z, u, idx, 1.0, "float32", "float32")
        assert np.isfinite(loss[:2]).all() and loss[2] == np.inf and np.isnan(loss[3:5]).all() and loss[5] == 0
        assert np.isfinite(dz[:3]).all() and np.isnan(dz[3:5]).all() and not dz[5].any()


@pytest.mark.parametrize("size", [1, 30, 700, 3000, 1e5, 1e20])
def test_distillation_of_large_logits(tf, size):
    """Across the point where max * log2(e) / T no longer fits beside the terms."""
    rng = _rng(int(np.log(size)), 4)
    z = rng.normal(0, 1, (9, 1200)) * size + size * rng.choice([-1, 1], (9, 1))
    idx, u = _teacher(rng, 9, 1200, 7)
    z[np.arange(9)[:, None], idx] = z.max(-1, keepdims=True) - rng.uniform(0, 3, idx.shape)   # some q are not 0
    for t in (1.0, 0.7):
        _check_distillation(tf, z, u * min(size, 1e3), idx, t, "float32", "float32")


def test_distillation_ignores_rows_without_weight(tf):
    rng = _rng(8)
    z = rng.normal(0, 2, (4, 50))
    idx, u = _teacher(rng, 4, 50, 3)
    _, dz = _check_distillation(tf, z, u, idx, 1.0, "float16", "float32", np.array([0, 1, 0, -2], np.float32))
    assert not dz[0].any() and not dz[2].any()


# ---- the three in one model, through the tape ----------------------------------------------------------
def _model(ops, tokens, u, idx, scale):
    def loss(table, gamma, beta, w):
        e = ops.embedding_lookup(table, tokens, scale)
        h = ops.layer_norm(e, gamma, beta)
        logits = ops.matmul(h, w)
        return ops.sum(ops.distillation_loss(logits, u, idx, 2.0))
    return loss


def test_model_gradients_against_differences(tf):
    """table -> lookup -> layerNorm -> matMul -> distillationLoss -> sum; the tape's gradients against
    central differences of a float64 numpy model."""
    ops = tf.ops
    rng = _rng(11)
    tokens, vocab, width, classes, top = 24, 11, 16, 20, 3
    idx_t = _tokens(rng, tokens, vocab)
    idx_c, u = _teacher(rng, tokens, classes, top)
    idx_c[2, 1:], idx_c[4] = -1, -1
    values = [rng.normal(0, 1, s).astype(np.float32) for s in ([vocab, width], [width], [width], [width, classes])]
    u = u.astype(np.float32)

    def f64(table, gamma, beta, w):
        ok = (idx_t >= 0) & (idx_t < vocab)
        e = np.where(ok[:, None], table[np.where(ok, idx_t, 0)] * 1.5, 0)
        c = e - e.mean(-1, keepdims=True)
        h = c / np.sqrt((c * c).mean(-1, keepdims=True) + EPS) * gamma + beta
        return _distillation_reference(h @ w, u, idx_c, np.ones(tokens), 2.0)[0].sum()

    want = []
    for i, v in enumerate(values):
        g = np.zeros(v.shape)
        for at in np.ndindex(*v.shape):
            args = [a.astype(np.float64) for a in values]
            args[i][at] += 1e-5
            up = f64(*args)
            args[i][at] -= 2e-5
            g[at] = (up - f64(*args)) / 2e-5
        want.append(g)
    before = tf.ENGINE.numTensors
    tensors = [ops.tensor(v) for v in values]
    ti, tu, tc = ops.tensor(idx_t, dtype="int32"), ops.tensor(u), ops.tensor(idx_c, dtype="int32")
    value, grads = ops.value_and_grads(_model(ops, ti, tu, tc, 1.5))(tensors)
    scale = [np.abs(w).max() for w in want]
    assert abs(float(value.dataSync()[0]) - f64(*[v.astype(np.float64) for v in values])) <= 1e-5 * tokens * 10
    for g, w, s in zip(grads, want, scale):
        assert np.abs(g.dataSync().reshape(w.shape) - w).max() <= 1e-4 * s
    for t in grads + [value, ti, tu, tc] + tensors:
        t.dispose()
    assert tf.ENGINE.numTensors == before


def test_layer_norm_over_several_axes_and_in_half_storage_mode(tf):
    ops, bk = tf.ops, tf.ENGINE.backend
    rng = _rng(13)
    x = rng.normal(0, 1, (3, 5, 4, 6)).astype(np.float32)
    g, b = rng.normal(1, 0.2, (2, 4, 6)).astype(np.float32)
    want, off, _, _ = _ln_reference(x.reshape(15, 24), g.reshape(-1), b.reshape(-1))
    y = ops.layer_norm(ops.tensor(x), ops.tensor(g), ops.tensor(b), axis=[2, -1])
    assert y.shape == [3, 5, 4, 6]
    _within(y.dataSync(), want, off)
    try:
        bk.setActivationStorage("float16")
        y = ops.layer_norm(ops.tensor(x), ops.tensor(g), ops.tensor(b), axis=[2, 3])
        e = ops.embedding_lookup(ops.tensor(x.reshape(60, 6)), ops.tensor([3, 59], dtype="int32"))
    finally:
        bk.setActivationStorage("float32")
    assert bk._rec(y.dataId)["dtype"] == "float16" and bk._rec(e.dataId)["dtype"] == "float16"
    _within(y.dataSync(), want, off + _half_step(want, "float16"))
    assert np.array_equal(e.dataSync().reshape(2, 6), _as_stored(x.reshape(60, 6)[[3, 59]], "float16"))


# ---- the calls around them ---------------------------------------------------------------------------
def _step(tf, t):
    """One training step's worth of backend calls on tensors t; returns every output."""
    bk = tf.ENGINE.backend
    e = bk.embeddingLookup(t["table"], t["tokens"], 2.0)
    y, stats = bk.layerNorm(e, t["gamma"], t["beta"], EPS, True)
    loss, ls = bk.distillationLoss(y, t["u"], t["classes"], 2.0)
    dy = bk.distillationLossBackprop(t["dloss"], y, t["u"], t["classes"], ls, 2.0)
    dx, dg, db = bk.layerNormBackprop(dy, e, t["gamma"], stats)
    return [e, y, loss, dy, dx, dg, db, bk.embeddingLookupBackprop(dx, t["tokens"], t["table"].shape[0], 2.0)]


def _step_inputs(tf, seed, tokens=300, vocab=70, width=136, top=4):
    rng = _rng(seed)
    idx, u = _teacher(rng, tokens, width, top)
    a = {"table": rng.normal(0, 1, (vocab, width)), "gamma": rng.normal(1, 0.1, width), "beta": rng.normal(0, 0.1, width),
         "u": u, "dloss": rng.uniform(0, 1, tokens)}
    return dict({k: v.astype(np.float32) for k, v in a.items()}, tokens=_tokens(rng, tokens, vocab), classes=idx)


def _upload(tf, arrays):
    return {k: tf.ops.tensor(v, dtype="int32" if v.dtype == np.int32 else "float32") for k, v in arrays.items()}


@pytest.mark.parametrize("tokens", [300, 5000, 70000])
def test_captured_graph_replays_on_new_inputs(tf, tokens):
    bk = tf.ENGINE.backend
    first, second, third = (_step_inputs(tf, s, tokens) for s in (1, 2, 3))
    t, other = _upload(tf, first), _upload(tf, second)
    bk.graphBegin()
    outs = _step(tf, t)
    graph = bk.graphEnd()
    bk.graphBegin()
    outs2 = _step(tf, other)   # a second graph: its workspaces are its own
    graph2 = bk.graphEnd()
    for arrays in (first, third, second):
        for k, v in arrays.items():
            bk.write(t[k].dataId, v)
        bk.graphLaunch(graph)
        bk.graphLaunch(graph2)
        bk.graphLaunch(graph)
        want, want2 = _step(tf, _upload(tf, arrays)), _step(tf, other)
        for a, b in zip(outs + outs2, want + want2):
            assert np.array_equal(a.dataSync(), b.dataSync())
    bk.graphDestroy(graph)
    bk.graphDestroy(graph2)


def test_captured_clusters(tf):
    bk = tf.ENGINE.backend
    rng = _rng(31)
    x, dy = rng.normal(0, 1, (2, 200, 20004)).astype(np.float32)
    g = rng.normal(1, 0.2, 20004).astype(np.float32)
    tx, td, tg = (tf.ops.tensor(v) for v in (x, dy, g))

    def step():
        y, stats = bk.layerNorm(tx, tg, tg, EPS, True)
        return [y, stats, *bk.layerNormBackprop(td, tx, tg, stats)]
    bk.graphBegin()
    outs = step()
    graph = bk.graphEnd()
    for v in (x, dy):
        bk.write(tx.dataId, v)
        bk.graphLaunch(graph)
        for a, b in zip(outs, step()):
            assert np.array_equal(a.dataSync(), b.dataSync())
    bk.graphDestroy(graph)


@pytest.mark.parametrize("option", ["pdl", "debug_sync"])
def test_launch_options_do_not_change_results(tf, option):
    bk = tf.ENGINE.backend
    t = _upload(tf, _step_inputs(tf, 41, 4000))
    want = [o.dataSync() for o in _step(tf, t)]
    bk.setOption(option, 1)
    try:
        for _ in range(3):
            outs = _step(tf, t)
            soft = bk.softmax(outs[-1])      # a kernel of the library behind the last one
            got = [o.dataSync() for o in outs]
            for a, b in zip(got, want):
                assert np.array_equal(a, b)
            e = np.exp(got[-1].reshape(70, -1).astype(np.float64) - got[-1].reshape(70, -1).max(-1, keepdims=True))
            assert np.abs(soft.dataSync().reshape(70, -1) - e / e.sum(-1, keepdims=True)).max() < 1e-6
    finally:
        bk.setOption(option, 0)


def test_guard_patterns_stay_intact(tf):
    bk = tf.ENGINE.backend
    bk.setOption("debug_canary", 1)
    try:
        for tokens, vocab, width in [(7, 5, 33), (65, 20, 1001), (1030, 3, 64), (70000, 40, 6), (3, 4, 20003),
                                     (200, 9, 9001), (150, 7, 16400), (31, 5, 3001), (2000, 11, 130)]:
            outs = tf.ENGINE.tidy(lambda: _step(tf, _upload(tf, _step_inputs(tf, width, tokens, vocab, width, 3))))
            for o in outs:
                o.dispose()
            bk.sync()   # an overwritten guard would be reported here
    finally:
        bk.setOption("debug_canary", 0)


def _filled(bk, shape, storage, fill):
    import torch
    t = bk.registerStored(list(shape), storage)
    view = torch.as_tensor(bk.deviceArray(t), device="cuda")
    fill(view)
    return t, view


@pytest.mark.parametrize("rows,width", [(2100000, 1024), (2145003, 1003), (66000, 33000)])
def test_layer_norm_offsets_past_32_bits(tf, rows, width):
    import torch
    bk = tf.ENGINE.backend
    torch.manual_seed(3)
    x, vx = _filled(bk, (rows, width), "float16", lambda v: v.normal_())
    g = _rng(1).normal(1, 0.2, width).astype(np.float32)
    torch.cuda.synchronize()
    y, stats = bk.layerNorm(x, tf.ops.tensor(g), None, EPS, True, "float16")
    bk.sync()
    vy, vs = (torch.as_tensor(bk.deviceArray(t), device="cuda") for t in (y, stats))
    dx, dg, db = bk.layerNormBackprop(y, x, tf.ops.tensor(g), stats)
    bk.sync()
    vd = torch.as_tensor(bk.deviceArray(dx), device="cuda")
    for rows_at in (slice(0, 3), slice(rows // 2, rows // 2 + 3), slice(rows - 3, rows)):
        xs, ys, ss, ds = (v[rows_at].float().cpu().numpy() for v in (vx, vy, vs, vd))
        want, off, _, _ = _ln_reference(xs, g, np.zeros(width, np.float32))
        _within(ys, want, off + _half_step(want, "float16"))
        (want, off), _, _ = _ln_backward_reference(ys, xs, g, ss)
        _within(ds, want, off)
    # dbeta: a column's sum of two million terms; its error is far below the share of one row that a wrong
    # offset would lose or count twice, taken over all columns
    total = sum(vy[i:i + 10000].double().sum(0) for i in range(0, rows, 10000)).cpu().numpy()
    assert np.abs(db.dataSync() - total).max() <= CHAIN * U * rows
    for t in (x, y, stats, dx, dg, db):
        t.dispose()


def test_embedding_offsets_past_32_bits(tf):
    import torch
    bk = tf.ENGINE.backend
    rows, width = 2100000, 1024
    table, vt = _filled(bk, (rows, width), "float16", lambda v: v.normal_())
    idx = np.array([rows - 1, 0, 2097152, rows, 2097151, rows - 1], np.int32)
    torch.cuda.synchronize()
    out = bk.embeddingLookup(table, tf.ops.tensor(idx, dtype="int32"), 1.0, "float16").dataSync().reshape(6, width)
    for k in (0, 1, 2, 4, 5):
        assert np.array_equal(out[k], vt[int(idx[k])].float().cpu().numpy())
    assert not out[3].any()
    small = bk.registerStored([50, width], "float16", _rng(1).normal(0, 1, 50 * width).astype(np.float32))
    many, vi = _filled(bk, (rows,), "int32", lambda v: v.copy_(torch.arange(rows, device="cuda") % 50))
    torch.cuda.synchronize()
    wide = bk.embeddingLookup(small, many, 1.0, "float16")
    bk.sync()
    vw = torch.as_tensor(bk.deviceArray(wide), device="cuda")
    assert torch.equal(vw[-100:], vw[:50].repeat(2, 1)) and torch.equal(vw[:50].cpu().float().reshape(-1), torch.from_numpy(small.dataSync()))
    # gradients: of a table past 32 bits from few tokens, of a small one from rows past 32 bits (all ones: counts)
    dy = tf.ops.tensor(np.arange(6, dtype=np.float32)[:, None] * np.ones((6, width), np.float32))
    dt = bk.embeddingLookupBackprop(dy, tf.ops.tensor(idx, dtype="int32"), rows, 1.0)
    bk.sync()
    vd = torch.as_tensor(bk.deviceArray(dt), device="cuda")
    want = {rows - 1: 5.0, 0: 1.0, 2097152: 2.0, 2097151: 4.0}
    for r, v in want.items():
        assert bool((vd[r] == v).all())
    assert float(vd.sum(dtype=torch.float64)) == sum(want.values()) * width
    dt.dispose()
    vw.fill_(1.0)
    torch.cuda.synchronize()
    counts = bk.embeddingLookupBackprop(wide, many, 50, 1.0)
    assert np.array_equal(counts.dataSync().reshape(50, width), np.full((50, width), rows // 50, np.float32))
    for t in (table, wide, many, counts):
        t.dispose()


def test_distillation_offsets_past_32_bits(tf):
    import torch
    bk = tf.ENGINE.backend
    rows, classes, top = 16401, 131073, 4
    z, vz = _filled(bk, (rows, classes), "float16", lambda v: v.normal_())
    rng = _rng(5)
    idx = rng.integers(0, classes, (rows, top)).astype(np.int32)
    u = rng.normal(0, 2, (rows, top)).astype(np.float32)
    dloss = rng.uniform(0.5, 1, rows).astype(np.float32)
    tu, ti = tf.ops.tensor(u), tf.ops.tensor(idx, dtype="int32")
    torch.cuda.synchronize()
    loss, stats = bk.distillationLoss(z, tu, ti, 1.0)
    dz = bk.distillationLossBackprop(tf.ops.tensor(dloss), z, tu, ti, stats, 1.0)
    bk.sync()
    vd = torch.as_tensor(bk.deviceArray(dz), device="cuda")
    got = loss.dataSync()
    for at in (slice(0, 2), slice(rows // 2, rows // 2 + 2), slice(rows - 2, rows)):
        want, off, dwant, doff, _ = _distillation_reference(vz[at].float().cpu().numpy(), u[at], idx[at], dloss[at], 1.0)
        _within(got[at], want, off)
        _within(vd[at].cpu().numpy(), dwant, doff)
    for t in (z, loss, stats, dz):
        t.dispose()


def test_two_contexts_at_once(tf):
    """Each context has its own stream and workspaces: interleaved steps give the same bits as alone."""
    tf.register_backend("cuda-second", 0)
    arrays = [_step_inputs(tf, s, 3000) for s in (21, 22)]
    try:
        results = []
        for repeat in range(2):
            sides = []
            for name, a in zip(("cuda", "cuda-second"), arrays):
                assert tf.set_backend(name)
                sides.append([name, _upload(tf, a), None])
            for _ in range(3):
                for side in sides:
                    tf.set_backend(side[0])
                    side[2] = _step(tf, side[1])
            for name, _, outs in sides:
                tf.set_backend(name)
                results.append([o.dataSync() for o in outs])
        for a, b in zip(results[:2], results[2:]):
            for x, y in zip(a, b):
                assert np.array_equal(x, y)
    finally:
        tf.set_backend("cuda")
        tf.ENGINE.removeBackend("cuda-second")


def test_zero_sizes(tf):
    bk = tf.ENGINE.backend
    z = lambda *s: tf.ops.tensor(np.zeros(s, np.float32), list(s))  # noqa: E731
    i = lambda *s: tf.ops.tensor(np.zeros(s, np.int32), list(s), "int32")  # noqa: E731
    y, s = bk.layerNorm(z(0, 8), z(8), z(8), EPS, True)
    assert y.shape == [0, 8] and s.shape == [0, 2]
    dx, dg, db = bk.layerNormBackprop(z(0, 8), z(0, 8), z(8), z(0, 2))
    assert dx.size == 0 and not dg.dataSync().any() and not db.dataSync().any() and dg.size == 8
    dx, dg, db = bk.layerNormBackprop(z(3, 0), z(3, 0), z(0), z(3, 2))
    assert dx.size == dg.size == 0
    assert bk.layerNorm(z(3, 0), z(0), z(0), EPS)[0].shape == [3, 0]
    assert bk.embeddingLookup(z(5, 4), i(0), 1.0).shape == [0, 4]
    assert not bk.embeddingLookup(z(0, 4), i(3), 1.0).dataSync().any()
    assert bk.embeddingLookup(z(5, 0), i(3), 1.0).shape == [3, 0]
    g = bk.embeddingLookupBackprop(z(0, 4), i(0), 6)
    assert g.shape == [6, 4] and not g.dataSync().any()
    assert bk.embeddingLookupBackprop(z(3, 4), i(3), 0).shape == [0, 4]
    assert bk.embeddingLookup(z(5, 4), tf.ops.scalar(2, "int32")).shape == [4]
    loss, st = bk.distillationLoss(z(0, 7), z(0, 2), i(0, 2))
    assert loss.shape == [0] and bk.distillationLossBackprop(z(0), z(0, 7), z(0, 2), i(0, 2), st).shape == [0, 7]
    loss, st = bk.distillationLoss(z(3, 0), z(3, 2), i(3, 2))
    assert not loss.dataSync().any()
    assert bk.distillationLossBackprop(z(3), z(3, 0), z(3, 2), i(3, 2), st).shape == [3, 0]


def test_refusals_leave_the_context_usable(tf):
    from tfjs_core_b200 import CudaError
    bk = tf.ENGINE.backend
    z = lambda *s: tf.ops.tensor(np.zeros(s, np.float32), list(s))  # noqa: E731
    i = lambda *s: tf.ops.tensor(np.zeros(s, np.int32), list(s), "int32")  # noqa: E731
    tensors = tf.ENGINE.numTensors
    calls = [
        lambda: bk.layerNorm(z(2, 8), z(7), None, EPS),
        lambda: bk.layerNorm(z(2, 8), None, z(9), EPS),
        lambda: bk.layerNorm(z(2, 8), None, None, -1.0),
        lambda: bk.layerNorm(z(2, 8), None, None, float("nan")),
        lambda: bk.layerNormBackprop(z(2, 7), z(2, 8), None, z(2, 2)),
        lambda: bk.layerNormBackprop(z(2, 8), z(2, 8), None, z(3, 2)),
        lambda: bk.distillationLoss(z(2, 8), z(2, 1025), i(2, 1025)),
        lambda: bk.distillationLoss(z(2, 8), z(2, 2), i(2, 2), 0.0),
        lambda: bk.distillationLoss(z(2, 8), z(2, 2), i(2, 2), float("inf")),
        lambda: bk.distillationLoss(z(2, 8), z(2, 2), i(2, 2), 1e-45),
        lambda: bk.distillationLossBackprop(z(3), z(2, 8), z(2, 2), i(2, 2), z(2, 4)),
        lambda: bk.distillationLossBackprop(z(2), z(2, 8), z(2, 2), i(2, 2), z(2, 3)),
        lambda: bk.layerNorm(bk.registerQuantized([2, 8], np.zeros(16), 1, 0), None, None, EPS),
        lambda: bk.registerStored([3], "float32", np.zeros(2)),
        lambda: bk.registerStored([3], "float16", np.zeros(4)),
    ]
    for call in calls:
        with pytest.raises(CudaError):
            tf.ENGINE.tidy(call)
    for call in (lambda: bk.layerNorm(z(), None, None, EPS), lambda: bk.embeddingLookup(z(3), i(2)),
                 lambda: bk.embeddingLookupBackprop(z(3, 4), i(2), 5), lambda: bk.distillationLoss(z(2, 8), z(3, 2), i(3, 2)),
                 lambda: bk.distillationLoss(z(2, 8), z(2, 2), i(2, 3)), lambda: bk.registerStored([2], "bool")):
        with pytest.raises(ValueError):
            tf.ENGINE.tidy(call)
    assert tf.ENGINE.numTensors == tensors   # a refused call leaves no output behind
    lib, ctx, a, s = bk._lib, bk._ctx, z(2, 8), z(2, 2)
    oid = bk._oid
    assert lib.tfjs_cuda_layer_norm(ctx, oid(a), 0, 0, oid(a), 0, 2, 8, EPS) == -1             # in place
    assert lib.tfjs_cuda_layer_norm(ctx, 10 ** 9, 0, 0, oid(a), 0, 2, 8, EPS) == -6            # no such tensor
    assert lib.tfjs_cuda_layer_norm(ctx, oid(a), 0, 0, oid(z(2, 8)), 0, -2, 8, EPS) == -1
    assert lib.tfjs_cuda_layer_norm(ctx, oid(a), 0, 0, oid(z(2, 8)), 0, 2 ** 40, 2 ** 30, EPS) == -1
    assert lib.tfjs_cuda_layer_norm_backprop(ctx, oid(a), oid(a), 0, 0, oid(z(2, 8)), 0, 0, 2, 8) == -1
    assert lib.tfjs_cuda_layer_norm_backprop(ctx, oid(a), oid(a), 0, oid(s), oid(a), 0, 0, 2, 8) == -1
    assert lib.tfjs_cuda_embedding_lookup(ctx, oid(a), oid(s), oid(z(2, 8)), 2, 2, 8, 1.0) == -1   # indices not int32
    assert lib.tfjs_cuda_embedding_lookup_backprop(ctx, oid(a), oid(i(2)), oid(a), 2, 2, 8, 1.0) == -1
    assert lib.tfjs_cuda_layer_norm(None, 1, 0, 0, 2, 0, 1, 1, EPS) == -1
    y, _ = bk.layerNorm(z(2, 8), None, None, EPS)
    assert not y.dataSync().any()


def test_device_arrays_are_views(tf):
    import torch
    bk = tf.ENGINE.backend
    a = _rng(17).normal(0, 1, (5, 6)).astype(np.float32)
    for storage in ("float32", "float16", "int32"):
        t = bk.registerStored([5, 6], storage)
        view = torch.as_tensor(bk.deviceArray(t), device="cuda")
        assert list(view.shape) == [5, 6] and str(view.dtype) == f"torch.{storage}"
        view.copy_(torch.from_numpy(a * 100))
        torch.cuda.synchronize()
        assert np.array_equal(t.dataSync().reshape(5, 6), (a * 100).astype(np.int32) if storage == "int32" else _as_stored(a * 100, storage))
    q = bk.registerQuantized([3], np.array([1, 2, 255], np.uint8), 0.5, 0.0)
    assert torch.as_tensor(bk.deviceArray(q), device="cuda").tolist() == [1, 2, 255]
    empty = bk.registerStored([0, 4], "float32")
    assert tuple(bk.deviceArray(empty).__cuda_array_interface__["shape"]) == (0, 4)
    t.dispose()
    with pytest.raises(RuntimeError, match="disposed"):
        bk.deviceArray(t)


def test_operands_of_other_storage_and_dtype_are_converted(tf):
    """bool and int32 tensors are float32 operands like everywhere else; float-stored indices truncate."""
    bk = tf.ENGINE.backend
    x = np.array([[1, 2, 3, 4], [5, 5, 5, 9]], np.int32)
    want, off, _, _ = _ln_reference(x.astype(np.float32), np.ones(4, np.float32), np.zeros(4, np.float32))
    y, _ = bk.layerNorm(tf.ops.tensor(x, dtype="int32"), None, None, EPS)
    _within(y.dataSync(), want, off)
    table = _rng(2).normal(0, 1, (4, 3)).astype(np.float32)
    out = bk.embeddingLookup(tf.ops.tensor(table), tf.ops.cast(tf.ops.tensor([1, 0, 1], dtype="bool"), "int32"))
    assert np.array_equal(out.dataSync().reshape(3, 3), table[[1, 0, 1]])


def test_single_rows_without_a_batch_axis(tf):
    ops = tf.ops
    rng = _rng(51)
    z, u = rng.normal(0, 2, 40).astype(np.float32), rng.normal(0, 2, 3).astype(np.float32)
    idx = np.array([3, 39, 7], np.int32)
    loss, (dz,) = ops.value_and_grads(lambda v: ops.distillation_loss(v, ops.tensor(u), ops.tensor(idx, dtype="int32"), 2.0))([ops.tensor(z)])
    want, off, dwant, doff, _ = _distillation_reference(z[None], u[None], idx[None], np.ones(1), 2.0)
    assert loss.shape == [] and dz.shape == [40]
    _within(loss.dataSync(), want, off)
    _within(dz.dataSync(), dwant, doff.reshape(1, 40))
    y, off, _, _ = _ln_reference(z[None], np.ones(40, np.float32), np.zeros(40, np.float32))
    _within(ops.layer_norm(ops.tensor(z)).dataSync(), y, off)
    assert ops.embedding_lookup(ops.tensor(z.reshape(10, 4)), ops.scalar(9, "int32")).dataSync().tolist() == z[36:].tolist()


def test_threads_with_contexts_of_their_own(tf):
    """Two host threads, each with its context on the same device, at sizes that need different shared memory."""
    import threading
    from tfjs_core_b200 import BackendCuda
    failures = []

    def work(widths, seed):
        try:
            bk = BackendCuda(0)
            lib, ctx = bk._lib, bk._ctx
            rng = _rng(seed)
            for repeat in range(40):
                for rows, width in widths:
                    arrays = [rng.normal(0, 1, (rows, width)).astype(np.float32), rng.normal(0, 1, (rows, width)).astype(np.float32)]
                    arrays.append(np.stack([arrays[1].mean(-1), 1 / np.sqrt(arrays[1].var(-1) + EPS)], -1).astype(np.float32))
                    ids = []
                    for a in arrays + [np.zeros((rows, width), np.float32), np.zeros(width, np.float32), np.zeros(width, np.float32)]:
                        ids.append(bk._new_id(a.shape, "float32"))
                        bk._check(lib.tfjs_cuda_tensor_write(ctx, ids[-1], np.ascontiguousarray(a).ctypes.data_as(C.c_void_p), a.nbytes))
                    bk._check(lib.tfjs_cuda_layer_norm_backprop(ctx, ids[0], ids[1], 0, ids[2], *ids[3:], rows, width))
                    out = np.empty((rows, width), np.float32)
                    bk._check(lib.tfjs_cuda_tensor_read(ctx, ids[3], out.ctypes.data_as(C.c_void_p), out.nbytes))
                    (want, off), _, _ = _ln_backward_reference(arrays[0], arrays[1], np.ones(width, np.float32), arrays[2])
                    _within(out, want, off)
                    bk._free_tmp(*ids)
            bk.dispose()
        except BaseException as e:   # seen by the main thread
            failures.append(repr(e)[:500])
    threads = [threading.Thread(target=work, args=a) for a in (([(2, 8192), (3, 4096)], 1), ([(64, 1020), (40, 2048)], 2))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not failures, failures


def test_upload_in_flight_is_waited_for(tf):
    bk = tf.ENGINE.backend
    n = 1 << 20
    host = C.c_void_p()
    assert bk._lib.tfjs_cuda_host_alloc(C.byref(host), n * 4) == 0
    arr = np.ctypeslib.as_array((C.c_float * n).from_address(host.value))
    arr[:] = _rng(5).normal(0, 1, n)
    t = tf.ops.tensor(np.zeros((n // 512, 512), np.float32))
    bk.writeAsync(t.dataId, host, n * 4)
    y, _ = bk.layerNorm(t, None, None, EPS)
    want, off, _, _ = _ln_reference(arr.reshape(-1, 512).copy(), np.ones(512, np.float32), np.zeros(512, np.float32))
    _within(y.dataSync(), want, off)
    bk._lib.tfjs_cuda_host_free(host)
