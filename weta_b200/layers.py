"""Fused layer ops on device storages: layer normalisation, forward and backward (include/weta_b200.h `wb_layer_norm_*`).

Tensors come as (storage, Layout, dtype), the way the backend's own methods take them; results are fresh contiguous
storages from the backend's arena unless `out` gives them.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

from .backend import B200Backend, BackendError, DeviceStorage
from .core import DType, Layout, WbView

_INVALID = 1  # WB_ERR_INVALID


def _declare(lib):
    if getattr(lib, "_wb_layers_declared", False):
        return
    P, V, i32, i64, f64 = ctypes.c_void_p, ctypes.POINTER(WbView), ctypes.c_int, ctypes.c_int64, ctypes.c_double
    sig = {
        "wb_layer_norm_fwd": ([P, V, i32, P, P, f64, P, P, P], i32),
        "wb_layer_norm_bwd_workspace": ([P, i64, i64, i32], i64),
        "wb_layer_norm_bwd": ([P, V, V, i32, P, P, P, P, P, P, P, i64], i32),
    }
    for name, (args, res) in sig.items():
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = args, res
    lib._wb_layers_declared = True


def _ptr(s: Optional[DeviceStorage]):
    return None if s is None else s.ptr


def _rows_cols(l: Layout, normalized_dims: int) -> Tuple[int, int]:
    rows = cols = 1
    for d, n in enumerate(l.shape):
        if d < l.ndim - normalized_dims:
            rows *= n
        else:
            cols *= n
    return rows, cols


def layer_norm_fwd(be: B200Backend, x: DeviceStorage, l: Layout, dt: int, normalized_dims: int, weight: Optional[DeviceStorage] = None,
                   bias: Optional[DeviceStorage] = None, eps: float = 1e-5,
                   out: Optional[Sequence[Optional[DeviceStorage]]] = None) -> Tuple[DeviceStorage, DeviceStorage, DeviceStorage]:
    """F::layer_norm (crates/weta-nn/src/functional.rs:183-195) over the last `normalized_dims` dims: (y, mean, rstd).

    `out` = (y, mean, rstd) writes there instead; mean and rstd may then be None, where no backward pass follows.
    """
    _declare(be.lib)
    v = l.view(x.ptr, dt)
    if out is None:
        if not 1 <= normalized_dims <= l.ndim or not DType.is_float(dt):
            out = (x, None, None)  # refused below, with the library's message
        else:
            rows, _ = _rows_cols(l, normalized_dims)
            out = (be.alloc(l.numel(), dt), be.alloc(rows, dt), be.alloc(rows, dt))
    y, mean, rstd = out
    be.check(be.lib.wb_layer_norm_fwd(be.handle, v, normalized_dims, _ptr(weight), _ptr(bias), eps, _ptr(y), _ptr(mean), _ptr(rstd)))
    return y, mean, rstd


def layer_norm_workspace(be: B200Backend, rows: int, cols: int, dt: int) -> DeviceStorage:
    """A workspace of the backward pass over [rows, cols]; calls that may run at the same time need one each."""
    _declare(be.lib)
    size = be.lib.wb_layer_norm_bwd_workspace(be.handle, rows, cols, dt)
    if size < 0:
        raise BackendError(_INVALID, f"layer norm of {rows} x {cols} values of dtype {dt}")
    return be.alloc(-(-size // DType.size(dt)), dt)


def layer_norm_bwd(be: B200Backend, x: DeviceStorage, lx: Layout, dy: DeviceStorage, ldy: Layout, dt: int, normalized_dims: int,
                   weight: Optional[DeviceStorage], mean: DeviceStorage, rstd: DeviceStorage,
                   out: Optional[Sequence[Optional[DeviceStorage]]] = None,
                   workspace: Optional[DeviceStorage] = None) -> Tuple[DeviceStorage, DeviceStorage, DeviceStorage]:
    """Its gradients (dx, dweight, dbias) from the forward pass's mean and rstd.

    `out` writes there instead, None leaves a gradient out.  Without a workspace one is taken from the backend's arena and
    given back after the call, which the arena orders on the backend's stream; a call that is captured into a CUDA
    graph brings its own and keeps it as long as the graph.
    """
    _declare(be.lib)
    vx, vg = lx.view(x.ptr, dt), ldy.view(dy.ptr, dt)
    if (out is None or workspace is None) and 1 <= normalized_dims <= lx.ndim and DType.is_float(dt):  # else: refused below
        rows, cols = _rows_cols(lx, normalized_dims)
        if out is None:
            out = (be.alloc(lx.numel(), dt), be.alloc(cols, dt), be.alloc(cols, dt))
        if workspace is None and cols and (out[1] is not None or out[2] is not None):
            workspace = layer_norm_workspace(be, rows, cols, dt)
    dx, dweight, dbias = out if out is not None else (None, None, None)
    size = 0 if workspace is None else workspace.length * DType.size(dt)
    be.check(be.lib.wb_layer_norm_bwd(be.handle, vx, vg, normalized_dims, _ptr(weight), _ptr(mean), _ptr(rstd), _ptr(dx), _ptr(dweight),
                                      _ptr(dbias), _ptr(workspace), size))
    return dx, dweight, dbias
