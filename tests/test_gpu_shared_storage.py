"""Tensors whose storage another library holds through deviceArray(): what it writes is seen by the next call,
also where the tensor is a weight, of which a repacked form is otherwise kept.  Truth: the same call on a fresh
tensor of the same values."""
import numpy as np
import pytest

from gpu_util import tf  # noqa: F401

pytestmark = pytest.mark.gpu


def _rng(seed):
    return np.random.Generator(np.random.PCG64(seed))


def _conv(x_shape, w_shape, stride, half=False):
    def call(tf, x, w):
        from tfjs_core_b200 import conv_util
        return tf.ENGINE.backend.fusedConv2d(x, w, conv_util.compute_conv2d_info(x_shape, w_shape, stride, 1, "same"))
    return x_shape, w_shape, call, half


CALLS = {
    "matMul": ((64, 96), (96, 128), lambda tf, x, w: tf.ops.matmul(x, w), False),
    "matMul, small": ((3, 5), (5, 2), lambda tf, x, w: tf.ops.matmul(x, w), False),
    "pointwise": _conv((1, 16, 16, 64), (1, 1, 64, 64), 1),
    "pointwise, half": _conv((1, 16, 16, 64), (1, 1, 64, 64), 1, True),
    "stem": _conv((1, 64, 64, 3), (3, 3, 3, 32), 2),
    "shifted patches": _conv((1, 16, 16, 32), (3, 3, 32, 64), 1),
    "gathered": _conv((1, 17, 17, 32), (3, 3, 32, 64), 2),
    "direct": _conv((1, 9, 9, 2), (3, 3, 2, 5), 1),
}


@pytest.mark.parametrize("mode", ["3xtf32", "tf32"])
@pytest.mark.parametrize("name", list(CALLS))
def test_weights_written_through_the_array(tf, name, mode):
    import torch
    bk = tf.ENGINE.backend
    x_shape, w_shape, call, half = CALLS[name]
    rng = _rng(len(name))
    x = bk.registerStored(list(x_shape), "float16" if half else "float32", rng.normal(0, 1, x_shape).astype(np.float32))
    values = rng.normal(0, 1, (3,) + w_shape).astype(np.float32)
    before = bk.math_mode
    bk.setMathMode(mode)
    try:
        shared = tf.ops.tensor(values[0])
        call(tf, x, shared)                       # its repacked form is kept from here on
        view = torch.as_tensor(bk.deviceArray(shared), device="cuda")
        for v in (values[1], values[2], values[1]):
            view.copy_(torch.from_numpy(v))
            torch.cuda.synchronize()
            want = call(tf, x, tf.ops.tensor(v)).dataSync()
            assert np.array_equal(call(tf, x, shared).dataSync(), want)
        bk.graphBegin()
        out = call(tf, x, shared)
        graph = bk.graphEnd()
        for v in values[:2]:                      # a replay repacks what the storage holds then
            view.copy_(torch.from_numpy(v))
            torch.cuda.synchronize()
            bk.graphLaunch(graph)
            assert np.array_equal(out.dataSync(), call(tf, x, tf.ops.tensor(v)).dataSync())
        bk.graphDestroy(graph)
    finally:
        bk.setMathMode(before)


@pytest.mark.parametrize("dequant_in_gemm", [0, 1])
def test_quantised_weights_written_through_the_array(tf, dequant_in_gemm):
    import torch
    bk = tf.ENGINE.backend
    rng = _rng(5)
    q = rng.integers(0, 256, (2, 96, 128)).astype(np.uint8)
    a = rng.normal(0, 1, (64, 96)).astype(np.float32)
    x, shared = tf.ops.tensor(a), bk.registerQuantized([96, 128], q[0], 0.02, -2.5)
    bk.setOption("dequant_in_gemm", dequant_in_gemm)
    try:
        tf.ops.matmul(x, shared)
        view = torch.as_tensor(bk.deviceArray(shared), device="cuda")
        for v in (q[1], q[0]):
            view.copy_(torch.from_numpy(v))
            torch.cuda.synchronize()
            w = v.astype(np.float64) * 0.02 - 2.5
            got = tf.ops.matmul(x, shared).dataSync().reshape(64, 128)
            # 3xTF32: products off by 2^-21 of themselves, 96 float32 additions
            assert np.all(np.abs(got - a.astype(np.float64) @ w) <= (2.0 ** -21 + 104 * 2.0 ** -24) * (np.abs(a) @ np.abs(w)))
    finally:
        bk.setOption("dequant_in_gemm", 0)


@pytest.mark.parametrize("which", ["depthwise", "pointwise"])
def test_separable_filters_written_through_the_array(tf, which):
    """An infinite tap that arrives through the array takes effect inside the image alone, as one from the host."""
    import torch
    from tfjs_core_b200 import conv_util
    bk = tf.ENGINE.backend
    rng = _rng(6)
    x = tf.ops.tensor(rng.uniform(0.5, 1, (1, 16, 16, 32)).astype(np.float32))
    wd, wp = rng.uniform(0.1, 0.5, (3, 3, 32, 1)).astype(np.float32), rng.uniform(0.1, 0.5, (1, 1, 32, 64)).astype(np.float32)
    ci = conv_util.compute_conv2d_info([1, 16, 16, 32], [3, 3, 32, 1], 1, 1, "same", None, True)
    before = bk.math_mode
    bk.setMathMode("tf32")
    try:
        td, tp = tf.ops.tensor(wd), tf.ops.tensor(wp)
        bk.fusedSeparableConv2d(x, td, tp, ci)
        shared, new = (td, wd.copy()) if which == "depthwise" else (tp, wp.copy())
        new.reshape(-1)[0] = np.inf if which == "depthwise" else 0.75
        view = torch.as_tensor(bk.deviceArray(shared), device="cuda")
        view.copy_(torch.from_numpy(new))
        torch.cuda.synchronize()
        fresh = tf.ops.tensor(new)
        want = bk.fusedSeparableConv2d(x, *((fresh, tp) if which == "depthwise" else (td, fresh)), ci).dataSync()
        got = bk.fusedSeparableConv2d(x, td, tp, ci).dataSync()
        assert np.array_equal(got, want, equal_nan=True)
        if which == "depthwise":   # the tap at (0, 0) lies outside the image for the first row and column only
            hit = np.isinf(got.reshape(16, 16, 64)[:, :, 0])
            assert hit[1:, 1:].all() and not hit[0].any() and not hit[:, 0].any()
    finally:
        bk.setMathMode(before)


def test_a_shared_quantised_tensor_that_needs_decoding_cannot_be_captured(tf):
    bk = tf.ENGINE.backend
    q = _rng(7).integers(0, 256, (5, 3)).astype(np.uint8)
    x, w = tf.ops.tensor(np.ones((2, 5), np.float32)), bk.registerQuantized([5, 3], q, 0.5, -1.0)
    want = tf.ops.matmul(x, w).dataSync()
    bk.deviceArray(w)
    bk.graphBegin()
    try:
        with pytest.raises(NotImplementedError, match="shared"):
            tf.ops.matmul(x, w)
    finally:
        bk.graphDestroy(bk.graphEnd())
    assert np.array_equal(tf.ops.matmul(x, w).dataSync(), want)
