"""CPU-only: layer norm and the many-tensor optimizer refuse storages of another element type, however long they are."""
import pytest

from weta_b200 import layers, optim
from weta_b200.backend import BackendError, DeviceStorage
from weta_b200.core import DType, Layout


class NoLib:
    """Fails the test where a call gets as far as the library."""
    _wb_layers_declared = _wb_optim_declared = True

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


class NoBackend:
    defers, handle = False, None

    def __init__(self, dt=DType.F32, n=1 << 20):
        self.lib = NoLib()
        self.lib.wb_storage_dtype = lambda handle: dt
        self.lib.wb_storage_len = lambda handle: n
        self.lib.wb_storage_data = lambda handle: 1 << 32


def storage(dt, n=1 << 20):
    return DeviceStorage(0, NoBackend(dt, n))


NAMES = {DType.F32: "f32", DType.F64: "f64", DType.I64: "i64"}
OTHERS = [(DType.F32, DType.F64), (DType.F32, DType.I64), (DType.F64, DType.F32), (DType.F64, DType.I64)]


@pytest.mark.parametrize("dt,other", OTHERS)
@pytest.mark.parametrize("which", ["x", "weight", "bias", "y", "mean", "rstd"])
def test_forward(which, dt, other):
    s = {k: storage(other if k == which else dt) for k in ("x", "weight", "bias", "y", "mean", "rstd")}
    with pytest.raises(BackendError, match=f"{which} is of {NAMES[other]}, not {NAMES[dt]}"):
        layers.layer_norm_fwd(NoBackend(), s["x"], Layout.contiguous([4, 8]), dt, 1, s["weight"], s["bias"], out=(s["y"], s["mean"], s["rstd"]))


@pytest.mark.parametrize("dt,other", OTHERS)
@pytest.mark.parametrize("which", ["x", "dy", "weight", "mean", "rstd", "dx", "dweight", "dbias"])
def test_backward(which, dt, other):
    s = {k: storage(other if k == which else dt) for k in ("x", "dy", "weight", "mean", "rstd", "dx", "dweight", "dbias")}
    l = Layout.contiguous([4, 8])
    with pytest.raises(BackendError, match=f"{which} is of {NAMES[other]}, not {NAMES[dt]}"):
        layers.layer_norm_bwd(NoBackend(), s["x"], l, s["dy"], l, dt, 1, s["weight"], s["mean"], s["rstd"], out=(s["dx"], s["dweight"], s["dbias"]),
                              workspace=storage(dt))


def optimizer():
    o = optim.AdamMulti.__new__(optim.AdamMulti)
    o.be, o.lib, o.handle, o.params = NoBackend(), NoLib(), None, [storage(DType.F32, 10)]
    o.be.handle = 1
    o.lib.wb_adam_multi_state_len = lambda handle: 256
    return o


@pytest.mark.parametrize("other", [DType.F64, DType.I64])
@pytest.mark.parametrize("which", [0, 1])
def test_scalars_of_the_norm(which, other):
    out = [storage(DType.F32), storage(DType.F32)]
    out[which] = storage(other)
    with pytest.raises(BackendError, match=f"{('norm', 'clip factor')[which]} is of {NAMES[other]}, not f32"):
        optimizer().grad_norm(1.0, out=out)


@pytest.mark.parametrize("other", [DType.F64, DType.I64])
@pytest.mark.parametrize("which", [0, 1])
def test_moments_that_are_read_back(which, other):
    for rest in (storage(DType.F32), None):
        out = [rest, rest]
        out[which] = storage(other)
        with pytest.raises(BackendError, match=f"{'mv'[which]} is of {NAMES[other]}, not f32"):
            optimizer().read_state(out=out)


@pytest.mark.parametrize("other", [DType.F64, DType.I64])
def test_parameters_gradients_and_the_scale(other):
    with pytest.raises(BackendError, match="parameter 0 is not f32"):
        optim.AdamMulti(NoBackend(), [storage(other, 10)])
    with pytest.raises(BackendError, match="gradient 0 is not f32"):
        optimizer().set_grads([storage(other, 10)])
    with pytest.raises(BackendError, match="scale is not a storage of f32"):
        optimizer().step(1, storage(other, 1))


def test_the_wait_test_hook_refuses():
    import ctypes

    from weta_b200.backend import load_library

    f = load_library().wb_layer_norm_selftest_timeout
    f.argtypes, f.restype = [ctypes.c_void_p, ctypes.c_int], ctypes.c_int
    handle = ctypes.create_string_buffer(1 << 16)
    for args in ((None, 100), (handle, 0), (handle, -1), (handle, (1 << 20) + 1)):
        assert f(*args) == 1
