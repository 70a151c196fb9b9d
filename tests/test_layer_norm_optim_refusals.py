"""CPU-only: what the layer-norm and many-tensor Adam entry points refuse, with the status and before any device work.

The backend handle here is zeroed host memory and the pointers are made up: a refusal looks at neither."""
import ctypes

import pytest

from weta_b200 import layers, optim
from weta_b200.backend import BackendError, DeviceStorage, load_library
from weta_b200.core import DType, Layout

INVALID, UNSUPPORTED = 1, 2
BASE = 1 << 32  # a made-up, well aligned device address


@pytest.fixture(scope="module")
def lib():
    lib = load_library()
    layers._declare(lib)
    optim._declare(lib)
    return lib


@pytest.fixture(scope="module")
def handle():
    return ctypes.create_string_buffer(1 << 16)


def addr(i):
    return BASE + (i << 24)


def fwd(lib, handle, layout=Layout.contiguous([4, 8]), dt=DType.F32, nd=1, x=0, w=1, b=2, eps=1e-5, y=3, mean=4, rstd=5, raw=None):
    p = lambda i: None if i is None else addr(i)
    v = layout.view(addr(x), dt)
    if raw:
        raw(v)
    return lib.wb_layer_norm_fwd(handle, v, nd, p(w), p(b), eps, p(y), p(mean), p(rstd))


def negative_dim(v):
    v.shape[0] = -1


def nine_dims(v):
    v.ndim = 9


def null_data(v):
    v.data = None


def huge_rows(v):
    v.shape[0] = 1 << 60


def huge_cols(v):
    v.shape[1] = 1 << 31


@pytest.mark.parametrize("change,status", [
    (dict(dt=DType.I64), UNSUPPORTED), (dict(nd=0), INVALID), (dict(nd=3), INVALID), (dict(nd=-1), INVALID), (dict(y=None), INVALID),
    (dict(eps=-1e-5), INVALID), (dict(eps=float("nan")), INVALID), (dict(layout=Layout.contiguous([4, 0])), INVALID),
    (dict(layout=Layout.contiguous([0, 0])), INVALID), (dict(raw=negative_dim), INVALID), (dict(raw=nine_dims), INVALID),
    (dict(raw=null_data), INVALID), (dict(raw=huge_rows), INVALID), (dict(raw=huge_cols), INVALID), (dict(y=0), INVALID),
    (dict(y=1), INVALID), (dict(mean=3), INVALID), (dict(mean=4, rstd=4), INVALID), (dict(y=2), INVALID)])
def test_forward_refuses(lib, handle, change, status):
    assert fwd(lib, handle, **change) == status
    assert lib.wb_last_error()


def test_forward_refuses_null_handle_view_and_unaligned_pointers(lib, handle):
    v = Layout.contiguous([4, 8]).view(addr(0), DType.F32)
    assert lib.wb_layer_norm_fwd(None, v, 1, None, None, 1e-5, addr(3), None, None) == INVALID
    assert lib.wb_layer_norm_fwd(handle, None, 1, None, None, 1e-5, addr(3), None, None) == INVALID
    for args in ((addr(1) + 2, None, addr(3)), (None, addr(2) + 1, addr(3)), (None, None, addr(3) + 2)):
        assert lib.wb_layer_norm_fwd(handle, v, 1, args[0], args[1], 1e-5, args[2], None, None) == INVALID
    # an output inside the reach of a negative stride
    back = Layout([4, 8], [-8, 1], 24).view(addr(0), DType.F32)
    assert lib.wb_layer_norm_fwd(handle, back, 1, None, None, 1e-5, addr(0), None, None) == INVALID


def test_no_rows_are_no_work(lib, handle):
    assert fwd(lib, handle, layout=Layout.contiguous([0, 8])) == 0


def bwd(lib, handle, lx=Layout.contiguous([4, 8]), lg=Layout.contiguous([4, 8]), dt=DType.F32, dg=DType.F32, nd=1, mean=3, rstd=4, dx=5, dw=6, db=7,
        ws=8, size=1 << 20):
    p = lambda i: None if i is None else addr(i)
    return lib.wb_layer_norm_bwd(handle, lx.view(addr(0), dt), lg.view(addr(1), dg), nd, addr(2), p(mean), p(rstd), p(dx), p(dw), p(db), p(ws), size)


@pytest.mark.parametrize("change,status", [
    (dict(dg=DType.F64), INVALID), (dict(dt=DType.I64, dg=DType.I64), UNSUPPORTED), (dict(lg=Layout.contiguous([4, 9])), INVALID),
    (dict(lg=Layout.contiguous([32])), INVALID), (dict(mean=None), INVALID), (dict(rstd=None), INVALID), (dict(ws=None), INVALID),
    (dict(size=63), INVALID), (dict(size=-1), INVALID), (dict(dx=0), INVALID), (dict(dx=1), INVALID), (dict(dw=2), INVALID),
    (dict(dw=3), INVALID), (dict(db=6), INVALID), (dict(ws=0), INVALID), (dict(ws=4), INVALID), (dict(ws=5), INVALID), (dict(nd=3), INVALID)])
def test_backward_refuses(lib, handle, change, status):
    assert bwd(lib, handle, **change) == status


def test_backward_workspace_refuses(lib, handle):
    f = lib.wb_layer_norm_bwd_workspace
    assert f(None, 4, 8, 0) == -1
    for rows, cols, dt in ((-1, 8, 0), (4, 0, 0), (4, 1 << 31, 0), (4, 8, 2), (4, 8, -1)):
        assert f(handle, rows, cols, dt) == -1
    assert f(handle, 0, 8, 0) == 0
    assert f(handle, 4, 8, 1) == 2 * f(handle, 4, 8, 0) > 0
    v = Layout.contiguous([4, 8]).view(addr(0), DType.F32)
    g = Layout.contiguous([4, 8]).view(addr(1), DType.F32)
    assert lib.wb_layer_norm_bwd(handle, v, g, 1, None, addr(3), addr(4), None, addr(6), None, addr(8) + 4, 1 << 20) == INVALID


def test_state_bytes(lib):
    def size(lens, bits):
        return lib.wb_adam_multi_state_bytes((ctypes.c_int64 * max(1, len(lens)))(*lens), len(lens), bits)

    assert size([1, 256, 257, 0], 32) == 8 * (256 + 256 + 512)
    assert size([1, 256, 257, 0], 8) == 2 * 1024 + 8 * 4
    assert size([0], 32) == 0
    for lens, bits in (([], 32), ([-1], 32), ([1], 16), ([1], 0), ([1 << 40, 1 << 40], 8), ([(1 << 63) - 1], 8)):
        assert size(lens, bits) == -1
    assert lib.wb_adam_multi_state_bytes(None, 1, 32) == -1


def create(lib, handle, tensors, bits=32, state=addr(9), size=1 << 22):
    arr = (optim.WbAdamTensor * max(1, len(tensors)))(*[optim.WbAdamTensor(p, n, 0, 0) for p, n in tensors])
    out = ctypes.c_void_p()
    return lib.wb_adam_multi_create(handle, arr, len(tensors), bits, state, size, 0, ctypes.byref(out))


@pytest.mark.parametrize("tensors,change,status", [
    ([], {}, INVALID), ([(addr(0), 10)], dict(bits=16), UNSUPPORTED), ([(None, 10)], {}, INVALID), ([(addr(0), -1)], {}, INVALID),
    ([(addr(0) + 2, 10)], {}, INVALID), ([(addr(0), 10)], dict(state=None), INVALID), ([(addr(0), 10)], dict(size=2047), INVALID),
    ([(addr(0), 10)], dict(state=addr(9) + 8), INVALID), ([(addr(0), 10), (addr(0), 10)], {}, INVALID),
    ([(addr(0) + 36, 10), (addr(1), 3), (addr(0), 10)], {}, INVALID), ([(addr(9) + 2044, 1)], {}, INVALID)])
def test_create_refuses(lib, handle, tensors, change, status):
    assert create(lib, handle, tensors, **change) == status


def test_null_handles(lib, handle):
    arr = (optim.WbAdamTensor * 1)(optim.WbAdamTensor(addr(0), 4, 0, 0))
    out = ctypes.c_void_p()
    assert lib.wb_adam_multi_create(None, arr, 1, 32, addr(9), 1 << 20, 0, ctypes.byref(out)) == INVALID
    assert lib.wb_adam_multi_create(handle, None, 1, 32, addr(9), 1 << 20, 0, ctypes.byref(out)) == INVALID
    assert lib.wb_adam_multi_create(handle, arr, 1, 32, addr(9), 1 << 20, 0, None) == INVALID
    assert lib.wb_adam_multi_destroy(None) == 0
    assert lib.wb_adam_multi_state_len(None) == -1 and lib.wb_adam_multi_offset(None, 0) == -1
    assert lib.wb_adam_multi_set_grads(None, None, 1) == INVALID
    assert lib.wb_adam_multi_grad_norm(None, 1.0, addr(1), None) == INVALID
    assert lib.wb_adam_multi_step(None, None, 1, 1.0, None) == INVALID
    assert lib.wb_adam_multi_read_state(None, addr(1), None) == INVALID


class FakeLib:
    """Fails the test where a call gets as far as the library."""
    _wb_layers_declared = _wb_optim_declared = True

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


class FakeBackend:
    lib, handle, defers = FakeLib(), None, False


def storage(n, dt=DType.F32):
    s = DeviceStorage.__new__(DeviceStorage)
    s.handle, s.backend, s.ptr, s._length, s._bytes = None, FakeBackend(), BASE, n, 0
    s.backend.lib = FakeLib()
    s.backend.lib.wb_storage_dtype = lambda handle: dt
    return s


@pytest.mark.parametrize("short", ["weight", "bias", "y", "mean", "rstd"])
@pytest.mark.parametrize("dt", [DType.F32, DType.F64])
def test_forward_refuses_short_storages(short, dt):
    need = dict(weight=8, bias=8, y=32, mean=4, rstd=4)
    s = {k: storage(n - (k == short), dt) for k, n in need.items()}
    with pytest.raises(BackendError, match=f"{short} holds"):
        layers.layer_norm_fwd(FakeBackend(), storage(32, dt), Layout.contiguous([4, 8]), dt, 1, s["weight"], s["bias"], out=(s["y"], s["mean"], s["rstd"]))


@pytest.mark.parametrize("short", ["weight", "mean", "rstd", "dx", "dweight", "dbias"])
@pytest.mark.parametrize("dt", [DType.F32, DType.F64])
def test_backward_refuses_short_storages(short, dt):
    need = dict(weight=8, mean=4, rstd=4, dx=32, dweight=8, dbias=8)
    s = {k: storage(n - (k == short), dt) for k, n in need.items()}
    l, x = Layout.contiguous([4, 8]), storage(32, dt)
    with pytest.raises(BackendError, match=f"{short} holds"):
        layers.layer_norm_bwd(FakeBackend(), x, l, x, l, dt, 1, s["weight"], s["mean"], s["rstd"], out=(s["dx"], s["dweight"], s["dbias"]),
                              workspace=storage(1 << 20, dt))


def test_a_storage_of_narrower_elements_is_too_short():
    s, l = storage(64, DType.F64), Layout.contiguous([4, 8])
    with pytest.raises(BackendError, match="weight holds 32 bytes, 64 are needed"):
        layers.layer_norm_fwd(FakeBackend(), s, l, DType.F64, 1, storage(8), None, out=(s, s, s))


def test_adam_refuses_storages_that_are_not_f32():
    o = optim.AdamMulti.__new__(optim.AdamMulti)
    o.be, o.lib, o.handle, o.params = FakeBackend(), FakeLib(), None, [storage(10)]
    with pytest.raises(BackendError, match="gradient 0 is not f32"):
        o.set_grads([storage(10, DType.F64)])
    with pytest.raises(BackendError, match="gradient 0 has 9"):
        o.set_grads([storage(9)])
    for s in (storage(1, DType.F64), storage(0)):
        with pytest.raises(BackendError, match="scale"):
            o.step(1, s)
    with pytest.raises(BackendError, match="norm"):
        o.grad_norm(1.0, out=(storage(1), storage(0)))
