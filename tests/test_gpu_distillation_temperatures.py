"""distillationLoss at temperatures whose square leaves the float32 range although the loss does not."""
import numpy as np
import pytest

from gpu_util import tf  # noqa: F401
from test_gpu_token_ops import _check_distillation, _rng, _teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("classes", [12, 1500, 40000])   # a warp a row, a block, a cluster
@pytest.mark.parametrize("t", [1e-30, 1e-25, 1e-15, 1e15])
def test_far_temperatures(tf, classes, t):
    rng = _rng(classes)
    z = rng.normal(0, 2, (5, classes))
    idx, u = _teacher(rng, 5, classes, 3)
    idx[3] = -1
    loss, _ = _check_distillation(tf, z, u, idx, t, "float32", "float32")
    assert (loss[[0, 1, 2, 4]] > 0).all() and loss[3] == 0


def test_one_class_and_a_square_that_overflows(tf):
    loss, dz = _check_distillation(tf, np.ones((2, 1)), np.ones((2, 1)), np.zeros((2, 1), np.int32), 1e20, "float32", "float32")
    assert not loss.any() and not dz.any()


def test_temperatures_without_a_finite_reciprocal_are_refused(tf):
    from tfjs_core_b200 import CudaError
    bk = tf.ENGINE.backend
    z, u, i = tf.ops.tensor(np.ones((2, 4), np.float32)), tf.ops.tensor(np.ones((2, 1), np.float32)), tf.ops.tensor(np.zeros((2, 1)), dtype="int32")
    for t in (3e-39, 4e-39, 1e-45, float("nan"), -1.0):
        with pytest.raises(CudaError, match="temperature"):
            tf.ENGINE.tidy(lambda: bk.distillationLoss(z, u, i, t))
