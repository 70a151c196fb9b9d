"""Fused layer ops on device storages: layer normalisation, forward and backward (include/weta_b200.h `wb_layer_norm_*`).

Tensors come as (storage, Layout, dtype), the way the backend's own methods take them; results are fresh contiguous
storages from the backend's arena unless `out` gives them.  All storages are checked for their element type, and those that
are taken whole for their length; a view is not checked against its storage, as in the backend's methods.
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


def _check(what: str, dt: int, *needs: Tuple[str, Optional[DeviceStorage], int]):
    """Refuses storages that hold fewer than so many elements of dtype `dt`, or elements of another type."""
    for name, s, n in needs:
        if s is not None and s.nbytes < n * DType.size(dt):
            raise BackendError(_INVALID, f"{what}: {name} holds {s.nbytes} bytes, {n * DType.size(dt)} are needed")
        if s is not None and s.dtype != dt:
            raise BackendError(_INVALID, f"{what}: {name} is of {DType.name(s.dtype)}, not {DType.name(dt)}")


def layer_norm_fwd(be: B200Backend, x: DeviceStorage, l: Layout, dt: int, normalized_dims: int, weight: Optional[DeviceStorage] = None,
                   bias: Optional[DeviceStorage] = None, eps: float = 1e-5,
                   out: Optional[Sequence[Optional[DeviceStorage]]] = None) -> Tuple[DeviceStorage, DeviceStorage, DeviceStorage]:
    """F::layer_norm (crates/weta-nn/src/functional.rs:183-195) over the last `normalized_dims` dims: (y, mean, rstd).

    `out` = (y, mean, rstd) writes there instead; mean and rstd may then be None, where no backward pass follows.
    """
    lib = be.lib
    if not hasattr(lib, "_wb_layers_declared"):
        _declare(lib)
    if be.defers:  # the outputs first: an operand that shares the storage of one gets another storage there
        out = None if out is None else be.for_writing(*out)
        x, weight, bias = be.for_reading(x, weight, bias)
    if 1 <= normalized_dims <= len(l.shape) and (dt == DType.F32 or dt == DType.F64):
        rows, cols = l.rows_cols(normalized_dims)
        if out is None:
            out = (be.alloc(rows * cols, dt), be.alloc(rows, dt), be.alloc(rows, dt))
        y, mean, rstd = out
        size = 4 if dt == DType.F32 else 8
        # the lengths in bytes as far as they are known: those that are not read as 0, and _check asks for them
        if (x.dtype != dt or (weight is not None and (weight._bytes < cols * size or weight.dtype != dt))
                or (bias is not None and (bias._bytes < cols * size or bias.dtype != dt))
                or (y is not None and (y._bytes < rows * cols * size or y.dtype != dt))
                or (mean is not None and (mean._bytes < rows * size or mean.dtype != dt))
                or (rstd is not None and (rstd._bytes < rows * size or rstd.dtype != dt))):
            _check("layer norm", dt, ("x", x, 0), ("weight", weight, cols), ("bias", bias, cols), ("y", y, rows * cols), ("mean", mean, rows),
                   ("rstd", rstd, rows))
    else:  # refused below, with the library's message
        y, mean, rstd = x, None, None
    status = lib.wb_layer_norm_fwd(be.handle, l.view(x.ptr, dt), normalized_dims, None if weight is None else weight.ptr,
                                   None if bias is None else bias.ptr, eps, None if y is None else y.ptr, None if mean is None else mean.ptr,
                                   None if rstd is None else rstd.ptr)
    if status:
        be.check(status)
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
    lib = be.lib
    if not hasattr(lib, "_wb_layers_declared"):
        _declare(lib)
    if be.defers:  # see layer_norm_fwd
        out = None if out is None else be.for_writing(*out)
        be.for_writing(workspace)
        x, dy, weight, mean, rstd = be.for_reading(x, dy, weight, mean, rstd)
    if 1 <= normalized_dims <= len(lx.shape) and (dt == DType.F32 or dt == DType.F64):  # else refused below
        rows, cols = lx.rows_cols(normalized_dims)
        if out is None:
            out = (be.alloc(rows * cols, dt), be.alloc(cols, dt), be.alloc(cols, dt))
        dx, dweight, dbias = out
        if workspace is None and cols and (dweight is not None or dbias is not None):
            workspace = layer_norm_workspace(be, rows, cols, dt)
        size = 4 if dt == DType.F32 else 8
        wide, tall = cols * size, rows * size
        if (x.dtype != dt or dy.dtype != dt or (mean is not None and (mean._bytes < tall or mean.dtype != dt))
                or (rstd is not None and (rstd._bytes < tall or rstd.dtype != dt))
                or (weight is not None and (weight._bytes < wide or weight.dtype != dt))
                or (dx is not None and (dx._bytes < rows * wide or dx.dtype != dt))
                or (dweight is not None and (dweight._bytes < wide or dweight.dtype != dt))
                or (dbias is not None and (dbias._bytes < wide or dbias.dtype != dt))):
            _check("layer norm's gradients", dt, ("x", x, 0), ("dy", dy, 0), ("mean", mean, rows), ("rstd", rstd, rows), ("weight", weight, cols),
                   ("dx", dx, rows * cols), ("dweight", dweight, cols), ("dbias", dbias, cols))
    else:
        dx, dweight, dbias = out if out is not None else (None, None, None)
    status = lib.wb_layer_norm_bwd(be.handle, lx.view(x.ptr, dt), ldy.view(dy.ptr, dt), normalized_dims, None if weight is None else weight.ptr,
                                   None if mean is None else mean.ptr, None if rstd is None else rstd.ptr, None if dx is None else dx.ptr, None if dweight is None else dweight.ptr,
                                   None if dbias is None else dbias.ptr, None if workspace is None else workspace.ptr,
                                   0 if workspace is None else workspace.nbytes)
    if status:
        be.check(status)
    return dx, dweight, dbias
