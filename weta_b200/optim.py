"""Adam / AdamW over many tensors at once: Python handle on `WbAdamMulti` (include/weta_b200.h)."""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

from .backend import B200Backend, BackendError, DeviceStorage
from .core import DType
from .trainer import WbAdamConfig


class WbAdamTensor(ctypes.Structure):
    _fields_ = [("theta", ctypes.c_void_p), ("len", ctypes.c_int64), ("no_decay", ctypes.c_int32), ("reserved", ctypes.c_int32)]


def _declare(lib):
    if getattr(lib, "_wb_optim_declared", False):
        return
    P, PP, i32, i64, f64 = ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p), ctypes.c_int, ctypes.c_int64, ctypes.c_double
    sig = {
        "wb_adam_multi_state_bytes": ([ctypes.POINTER(i64), i32, i32], i64),
        "wb_adam_multi_create": ([P, ctypes.POINTER(WbAdamTensor), i32, i32, P, i64, i32, PP], i32),
        "wb_adam_multi_destroy": ([P], i32),
        "wb_adam_multi_state_len": ([P], i64),
        "wb_adam_multi_offset": ([P, i32], i64),
        "wb_adam_multi_set_grads": ([P, PP, i32], i32),
        "wb_adam_multi_grad_norm": ([P, f64, P, P], i32),
        "wb_adam_multi_step": ([P, ctypes.POINTER(WbAdamConfig), i64, f64, P], i32),
        "wb_adam_multi_read_state": ([P, P, P], i32),
    }
    for name, (args, res) in sig.items():
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = args, res
    lib._wb_optim_declared = True


def _check_f32(name: str, s: Optional[DeviceStorage]):
    if s is not None and s.dtype != DType.F32:
        raise BackendError(1, f"{name} is of {DType.name(s.dtype)}, not f32")


class AdamMulti:
    """The optimizer of a list of f32 parameter storages (crates/weta-optim/src/lib.rs:178-239, 276-283).

    `state_bits` 32 keeps m and v as f32 and gives `wb_adam_step`'s bits; 8 keeps one byte each and a scale per 256
    elements.  `no_decay[i]` exempts tensor i from weight decay.  `state` is the moments' memory, an f32 storage of at least
    `state_bytes` bytes: its contents and the step count are all that a checkpoint needs; `keep_state` starts from what it
    holds.  Left out, it comes from the backend's arena, zeroed.
    """

    def __init__(self, backend: B200Backend, params: Sequence[DeviceStorage], state_bits: int = 32, no_decay: Optional[Sequence[bool]] = None,
                 lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0, decoupled: bool = False,
                 state: Optional[DeviceStorage] = None, keep_state: bool = False):
        self.be, self.lib, self.handle = backend, backend.lib, None
        _declare(self.lib)
        n = len(params)
        if backend.defers:
            backend.for_writing(*params, state)
        if no_decay is not None and len(no_decay) != n:
            raise BackendError(1, f"{len(no_decay)} no_decay flags for {n} tensors")
        self.params = list(params)
        lens = [p.length for p in params]
        for i, p in enumerate(params):
            if p.dtype != DType.F32:
                raise BackendError(1, f"parameter {i} is not f32")
        self.state_bytes = self.lib.wb_adam_multi_state_bytes((ctypes.c_int64 * max(n, 1))(*lens), n, state_bits)
        if state is None and self.state_bytes >= 0:
            if keep_state:
                raise BackendError(1, "keep_state without a state")
            state = backend.alloc(-(-self.state_bytes // 4), DType.F32)
        self.state = state
        arr = (WbAdamTensor * max(n, 1))(*[WbAdamTensor(p.ptr, k, int(bool(no_decay[i])) if no_decay is not None else 0, 0)
                                           for i, (p, k) in enumerate(zip(params, lens))])
        out = ctypes.c_void_p()
        backend.check(self.lib.wb_adam_multi_create(backend.handle, arr, n, state_bits, None if state is None else state.ptr,
                                                    0 if state is None else state.nbytes, int(keep_state), ctypes.byref(out)))
        self.handle = out.value
        self.config = WbAdamConfig(lr, betas[0], betas[1], eps, weight_decay, int(decoupled))  # may be changed between steps
        self._config = ctypes.byref(self.config)
        self._grads = None

    def close(self):
        if self.handle and self.be.handle:
            self.lib.wb_adam_multi_destroy(self.handle)
        self.handle = None

    def _open(self):
        if not self.be.handle:  # the library's handle points at the backend's memory
            raise BackendError(1, "the optimizer's backend is closed")

    def _call(self, entry, *args):
        self._open()
        self.be.check(entry(self.handle, *args))

    def _alloc(self, n):
        self._open()
        return self.be.alloc(n, DType.F32)

    def __del__(self):
        if getattr(self, "handle", None):
            self.close()

    @property
    def state_len(self) -> int:
        return self.lib.wb_adam_multi_state_len(self.handle)

    def offset(self, i: int) -> int:
        """Where tensor i's moments start, in elements of the state (and of `read_state`)."""
        return self.lib.wb_adam_multi_offset(self.handle, i)

    def set_grads(self, grads: Sequence[Optional[DeviceStorage]]):
        """The gradients of the following calls, in the parameters' order; None leaves a tensor and its state alone."""
        if self.be.defers:
            grads = self.be.for_keeping(*grads)
        for i, (g, p) in enumerate(zip(grads, self.params)):
            if g is not None and g.length != p.length:
                raise BackendError(1, f"gradient {i} has {g.length} elements, its parameter {p.length}")
            if g is not None and g.dtype != DType.F32:
                raise BackendError(1, f"gradient {i} is not f32")
        arr = (ctypes.c_void_p * max(len(grads), 1))(*[None if g is None else g.ptr for g in grads])
        self.be.check(self.lib.wb_adam_multi_set_grads(self.handle, arr, len(grads)))
        self._grads = list(grads)  # kept alive while the library holds their addresses

    def grad_norm(self, max_norm: float, out: Optional[Sequence[DeviceStorage]] = None) -> Tuple[DeviceStorage, DeviceStorage]:
        """(norm of all gradients, min(1, max_norm / (norm + 1e-6))) as device scalars; the second is `step`'s grad_scale."""
        norm, scale = out if out is not None else (self._alloc(1), self._alloc(1))
        if self.be.defers:
            self._open()
            self.be.for_writing(norm, scale)
        if norm.nbytes < 4 or (scale is not None and scale.nbytes < 4):
            raise BackendError(1, "an output of the norm holds no element")
        _check_f32("the norm", norm)
        _check_f32("the clip factor", scale)
        self._call(self.lib.wb_adam_multi_grad_norm, max_norm, norm.ptr, None if scale is None else scale.ptr)
        return norm, scale

    def step(self, t: int, grad_scale: Union[None, float, DeviceStorage] = None):
        """Step t, counted from 1; the gradients are multiplied by `grad_scale`, a number or a device scalar."""
        if self.be.defers:
            self._open()
            self.be.for_writing(*self.params, self.state)
            if hasattr(grad_scale, "ptr"):
                grad_scale, = self.be.for_reading(grad_scale)
        if grad_scale is None or isinstance(grad_scale, DeviceStorage):
            if grad_scale is not None and (grad_scale.length < 1 or grad_scale.dtype != DType.F32):
                raise BackendError(1, "the scale is not a storage of f32")
            host, device = 1.0, None if grad_scale is None else grad_scale.ptr
        else:
            host, device = float(grad_scale), None
        self._call(self.lib.wb_adam_multi_step, self._config, t, host, device)

    def read_state(self, out: Optional[Sequence[Optional[DeviceStorage]]] = None) -> Tuple[DeviceStorage, DeviceStorage]:
        """(m, v) as f32 storages of `state_len` elements: what the state stands for."""
        m, v = out if out is not None else (self._alloc(self.state_len), self._alloc(self.state_len))
        if self.be.defers:
            self._open()
            self.be.for_writing(m, v)
        need = 4 * self.state_len
        for name, s in (("m", m), ("v", v)):
            if s is not None and s.nbytes < need:
                raise BackendError(1, f"the moments take {need} bytes each, an output holds {s.nbytes}")
            _check_f32(name, s)
        self._call(self.lib.wb_adam_multi_read_state, None if m is None else m.ptr, None if v is None else v.ptr)
        return m, v
