"""layerNorm at widths whose dynamic shared memory stays within 48 KB while the kernel's static arrays take
the sum past it, each as the first call of its kernel in a fresh process (a call that asked for more before
would have raised the kernel's limit already)."""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# (what, rows, width, storage of dy, storage of x); no kernel twice in a process
PROCESSES = {
    "one of each kernel": [("forward", 3, 6135, "float32", "float32"), ("forward", 3, 12270, "float16", "float16"),
                           ("forward", 8, 98000, "float32", "float32"), ("backprop", 20, 16300, "float32", "float32"),
                           ("backprop", 20, 19568, "float32", "float16"), ("backprop", 20, 24448, "float16", "float16")],
    "four blocks a row": [("forward", 40, 49000, "float32", "float32")],
    "two blocks a row": [("forward", 80, 24500, "float32", "float32")],
}
U = 2.0 ** -24


def _run(cases):
    import tfjs_core_b200 as tf
    assert tf.set_backend("cuda")
    bk = tf.ENGINE.backend
    for what, rows, width, sd, sx in cases:
        rng = np.random.default_rng(width)
        stored = lambda s: bk.registerStored([rows, width], s, rng.normal(0, 1, (rows, width)).astype(np.float32))  # noqa: E731
        x = stored(sx)
        v = x.dataSync().reshape(rows, width).astype(np.float64)
        m, r = v.mean(-1, keepdims=True), 1 / np.sqrt(v.var(-1, keepdims=True) + 1e-5)
        n = (v - m) * r
        if what == "forward":
            y, stats = bk.layerNorm(x, None, None, 1e-5, True, "float32")
            # 256 roundings of the row's largest value in the mean, half as many of the scale
            tol = (256 * np.abs(v).max() + 136 * np.abs(n).max()) * U * r.max()
            assert np.abs(y.dataSync().reshape(rows, width) - n).max() <= tol, (rows, width)
            assert np.abs(stats.dataSync().reshape(rows, 2) - np.concatenate([m, r], -1)).max() <= 256 * U * np.abs(v).max()
        else:
            dy = stored(sd)
            d = dy.dataSync().reshape(rows, width).astype(np.float64)
            stats = tf.ops.tensor(np.concatenate([m, r], -1).astype(np.float32))
            dx, dg, db = bk.layerNormBackprop(dy, x, None, stats)
            want = r * (d - d.mean(-1, keepdims=True) - n * (d * n).mean(-1, keepdims=True))
            big = np.abs(d).max() * max(1.0, np.abs(n).max()) ** 2 * r.max()
            assert np.abs(dx.dataSync().reshape(rows, width) - want).max() <= 256 * U * big, (rows, width)
            assert np.abs(dg.dataSync() - (d * n).sum(0)).max() <= (rows + 8) * U * np.abs(d * n).sum(0).max()
            assert np.abs(db.dataSync() - d.sum(0)).max() <= (rows + 8) * U * np.abs(d).sum(0).max()


@pytest.mark.parametrize("cases", list(PROCESSES))
def test_widths_between_the_limits(cases):
    here = os.path.dirname(os.path.abspath(__file__))
    code = f"import sys; sys.path[:0] = [{os.path.dirname(here)!r}, {here!r}]; " \
           f"import test_gpu_shared_memory_opt_in as t; t._run(t.PROCESSES[{cases!r}])"
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr[-2000:]
