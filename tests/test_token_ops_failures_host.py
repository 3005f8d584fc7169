"""What the backend's methods of layerNorm, embeddingLookup and distillationLoss leave behind when a step of
them fails: nothing.  The library is a stand-in that counts its tensors and fails at a chosen call."""
import numpy as np
import pytest

from tfjs_core_b200 import _ffi, ops
from tfjs_core_b200.backend_cuda import BackendCuda, CudaError
from tfjs_core_b200.engine import ENGINE


class FakeLibrary:
    """Entry points as attributes: registrations, conversions and kernels are steps that can fail."""

    def __init__(self):
        self.live, self.next_id, self.steps, self.fail_at = set(), 0, 0, None

    def _step(self):
        self.steps += 1
        return -2 if self.steps == self.fail_at else 0

    def tfjs_cuda_ctx_create(self, device, out):
        out._obj.value = 1
        return 0

    def tfjs_cuda_tensor_register(self, ctx, out, rank, shape, dtype):
        rc = self._step()
        if rc == 0:
            self.next_id += 1
            self.live.add(self.next_id)
            out._obj.value = self.next_id
        return rc

    def tfjs_cuda_tensor_dispose(self, ctx, i):
        self.live.remove(i)   # a second disposal of the same id is an error here
        return 0

    def tfjs_cuda_last_error(self, ctx):
        return b"planted"

    def __getattr__(self, name):
        if name in ("tfjs_cuda_cast",) or name.startswith(("tfjs_cuda_layer", "tfjs_cuda_embedding", "tfjs_cuda_distillation")):
            return lambda *a: self._step()
        return lambda *a: 0   # context, options, writes, stream


@pytest.fixture()
def fake(monkeypatch):
    lib = FakeLibrary()
    monkeypatch.setattr(_ffi, "load", lambda: lib)
    prev = ENGINE.backendName
    ENGINE.registerBackend("fake-library-test", BackendCuda, 1000)
    assert ENGINE.setBackend("fake-library-test")
    yield lib, ENGINE.backend
    lib.fail_at = None
    ENGINE.removeBackend("fake-library-test")
    if prev:
        ENGINE.setBackend(prev)


def _t(*shape, dtype="int32"):   # int32 where float32 is wanted: each operand needs a conversion
    return ops.tensor(np.zeros(shape), list(shape), dtype)


METHODS = {
    "layerNorm": lambda b: (lambda x, g, s: b.layerNorm(x, g, s, 1e-5, True), [_t(2, 4), _t(4), _t(4)], 2),
    "layerNormBackprop": lambda b: (b.layerNormBackprop, [_t(2, 4), _t(2, 4), _t(4), _t(2, 2)], 3),
    "embeddingLookup": lambda b: (b.embeddingLookup, [_t(5, 4), _t(3, dtype="float32")], 1),
    "embeddingLookupBackprop": lambda b: (lambda d, i: b.embeddingLookupBackprop(d, i, 5), [_t(3, 4), _t(3, dtype="float32")], 1),
    "distillationLoss": lambda b: (b.distillationLoss, [_t(2, 4), _t(2, 1), _t(2, 1, dtype="float32")], 2),
    "distillationLossBackprop": lambda b: (b.distillationLossBackprop,
                                           [_t(2), _t(2, 4), _t(2, 1), _t(2, 1, dtype="float32"), _t(2, 4)], 1),
}


@pytest.mark.parametrize("name", list(METHODS))
def test_a_failed_step_leaves_nothing_behind(fake, name):
    lib, bk = fake
    call, operands, outputs = METHODS[name](bk)
    state = lambda: (set(lib.live), set(bk._data), ENGINE.numTensors, ENGINE.numBytes, ENGINE.numDataBuffers, len(ENGINE.tensorInfo))  # noqa: E731
    before = state()
    steps = 2 * len(operands) + outputs + 1   # a registration and a conversion an operand, the outputs, the kernel
    for lib.fail_at in range(1, steps + 1):
        lib.steps = 0
        with pytest.raises(CudaError, match="planted"):
            call(*operands)
        assert state() == before, lib.fail_at
    lib.fail_at, lib.steps = None, 0
    made = call(*operands)
    assert lib.steps == steps and len(lib.live) == len(before[0]) + outputs   # the conversions are gone
    for t in made if isinstance(made, tuple) else (made,):
        t.dispose()
    assert state() == before


def test_out_parameters_belong_to_their_call(fake):
    """Another thread's call may fill its out-parameter between this call and the reading of its own; played
    here by a library that makes that call before it returns."""
    lib, bk = fake
    t = ops.tensor(np.zeros(3, np.float32))
    inner, register, share = [], lib.tfjs_cuda_tensor_register, {bk._data[t.dataId]["id"]: 0x1000}

    def registering(ctx, out, *rest):
        rc = register(ctx, out, *rest)
        if not inner:
            inner.append(None)
            inner[0] = bk._new_id([2], "float32")
        return rc
    lib.tfjs_cuda_tensor_register = registering
    outer = bk._new_id([2], "float32")
    assert outer != inner[0] and {outer, inner[0]} <= lib.live
    other = ops.tensor(np.zeros(3, np.float32))
    share[bk._data[other.dataId]["id"]] = 0x2000
    nested = []

    def sharing(ctx, i, ptr, nbytes):
        ptr._obj.value = share[i]
        if not nested:
            nested.append(None)
            nested[0] = bk.deviceArray(other)
        return 0
    lib.tfjs_cuda_tensor_share = sharing
    arrays = bk.deviceArray(t), nested[0]
    assert [a.__cuda_array_interface__["data"][0] for a in arrays] == [0x1000, 0x2000]
