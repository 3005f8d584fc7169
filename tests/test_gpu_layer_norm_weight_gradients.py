"""dgamma and dbeta of layerNorm over more than 2^31 values, exactly.  dy is +-1 and x is +-1 or +-2, with a mean of
0 and a scale of 1 given as the statistics: every product is a whole number, every partial sum is below 2^24, and
float32 sums of them are exact in any order.  A row that is lost, counted twice or read at a wrong offset shifts
whole columns by 1 or more."""
import numpy as np
import pytest

from gpu_util import tf  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,width", [(2100000, 1024), (2145003, 1003), (66000, 33000), (2201, 1024), (1203, 1003), (61, 33000)])
def test_every_row_counts_once(tf, rows, width):
    import torch
    bk = tf.ENGINE.backend
    torch.manual_seed(rows)

    def filled(shape, storage, fill):
        t = bk.registerStored(list(shape), storage)
        view = torch.as_tensor(bk.deviceArray(t), device="cuda")
        for i in range(0, shape[0], 100000):
            fill(view[i:i + 100000])
        return t, view

    dy, vd = filled((rows, width), "float16", lambda v: v.random_(0, 2).mul_(2).sub_(1))
    x, vx = filled((rows, width), "float16", lambda v: v.random_(0, 4).sub_(1.75).round_().add_((v >= 0).to(v.dtype)))
    stats, _ = filled((rows, 2), "float32", lambda v: v.copy_(v.new_tensor([0.0, 1.0]).expand_as(v)))
    dgamma, dbeta = tf.ops.zeros([width]), tf.ops.zeros([width])
    torch.cuda.synchronize()
    assert set(vx[:1000].unique().tolist()) == {-2.0, -1.0, 1.0, 2.0} and set(vd[-1000:].unique().tolist()) == {-1.0, 1.0}
    rc = bk._lib.tfjs_cuda_layer_norm_backprop(bk._ctx, bk._oid(dy), bk._oid(x), 0, bk._oid(stats), 0, bk._oid(dgamma),
                                               bk._oid(dbeta), rows, width)
    assert rc == 0
    bk.sync()
    want_g, want_b = (torch.zeros(width, dtype=torch.float64, device="cuda") for _ in range(2))
    for i in range(0, rows, 20000):
        d = vd[i:i + 20000].double()
        want_b += d.sum(0)
        want_g += (d * vx[i:i + 20000].double()).sum(0)
    assert np.array_equal(dgamma.dataSync(), want_g.cpu().numpy()) and np.array_equal(dbeta.dataSync(), want_b.cpu().numpy())
    for t in (dy, x, stats, dgamma, dbeta):
        t.dispose()
