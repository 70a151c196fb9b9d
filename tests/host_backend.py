"""A backend in host memory with the calls that the fusing backend, `layers` and `optim` make: for CPU tests of which address
a call is given and what lies there at that moment.  Freed storages are filled with NaN."""
import ctypes
import itertools
import math

import numpy as np

from weta_b200.backend import BackendError, DeviceStorage
from weta_b200.core import BinaryOp, DType, Layout


def at(ptr, n):
    return np.ctypeslib.as_array(ctypes.cast(int(ptr), ctypes.POINTER(ctypes.c_float)), (n,))


class HostLib:
    _wb_layers_declared = _wb_optim_declared = True

    def __init__(self):
        self.memory, self.ids, self.calls = {}, itertools.count(1), []

        def ew_fused(handle, views, n_in, prog, n_instr, out_regs, out_ptrs, n_out, n):
            regs = []
            for p in prog[:n_instr]:
                if p.kind == 0:
                    regs.append(at(views[p.a].data + 4 * views[p.a].offset, n).copy())
                else:
                    assert (p.kind, p.op) == (2, BinaryOp.ADD)
                    regs.append(regs[p.a] + regs[p.b])
            for r, p in zip(out_regs[:n_out], out_ptrs[:n_out]):
                at(p, n)[:] = regs[r]
            return 0

        self.wb_ew_fused = ew_fused

    def new(self, n, dt):
        h = next(self.ids)
        self.memory[h] = (np.zeros(max(n, 1), DType.np(dt)), n, dt)
        return h

    def wb_storage_data(self, h):
        return self.memory[h][0].ctypes.data

    def wb_storage_len(self, h):
        return self.memory[h][1]

    def wb_storage_dtype(self, h):
        return self.memory[h][2]

    def wb_free(self, backend, h):
        self.memory[h][0].fill(np.nan if self.memory[h][2] != DType.I64 else -1)

    # the many-tensor optimizer: a step subtracts the gradient
    def wb_adam_multi_state_bytes(self, lens, n, bits):
        return sum(8 * (-(-k // 256) * 256) for k in lens[:n])

    def wb_adam_multi_create(self, backend, tensors, n, bits, state, size, keep, out):
        self.tensors = [(t.theta, t.len) for t in tensors[:n]]
        out._obj.value = next(self.ids)
        return 0

    def wb_adam_multi_destroy(self, h):
        self.calls.append("destroy")
        return 0

    def wb_adam_multi_set_grads(self, h, grads, n):
        self.grads = list(grads[:n])
        for g in self.grads:
            for p, k in self.tensors:
                if g is not None and p - 4 * k < g < p + 4 * k:
                    return 1
        return 0

    def wb_adam_multi_grad_norm(self, h, limit, norm, clip):
        at(norm, 1)[0] = math.sqrt(sum(float((at(g, k) ** 2).sum()) for g, (_, k) in zip(self.grads, self.tensors) if g))
        if clip:
            at(clip, 1)[0] = 1.0
        return 0

    def wb_adam_multi_step(self, h, cfg, t, scale, device_scale):
        self.calls.append("step")
        for g, (p, k) in zip(self.grads, self.tensors):
            if g:
                at(p, k)[:] -= at(g, k) * (at(device_scale, 1)[0] if device_scale else scale)
        return 0

    def wb_adam_multi_state_len(self, h):
        self.calls.append("state_len")
        return sum(-(-k // 256) * 256 for _, k in self.tensors)

    def wb_adam_multi_offset(self, h, i):
        self.calls.append("offset")
        return 0

    def wb_adam_multi_read_state(self, h, m, v):
        self.calls.append("read_state")
        return 0

    # layer norm: refuses overlapping operands, else notes the call and copies x to y (dy to dx)
    def _take(self, name, read, written, src, dst, n):
        for p, k in written:
            for q, j in read:
                if p and q and p < q + 4 * j and q < p + 4 * k:
                    return 1
        self.calls.append(name)
        if dst:
            at(dst, n)[:] = at(src, n)
        return 0

    def wb_layer_norm_fwd(self, backend, x, nd, w, b, eps, y, mean, rstd):
        n, cols = math.prod(x.shape), math.prod(x.shape[x.ndim - nd:x.ndim])
        src = x.data + 4 * x.offset
        return self._take("layer_norm_fwd", [(src, n), (w, cols), (b, cols)], [(y, n), (mean, n // cols), (rstd, n // cols)], src, y, n)

    def wb_layer_norm_bwd_workspace(self, backend, rows, cols, dt):
        return 64

    def wb_layer_norm_bwd(self, backend, x, dy, nd, w, mean, rstd, dx, dw, db, work, size):
        n, cols = math.prod(x.shape), math.prod(x.shape[x.ndim - nd:x.ndim])
        src = dy.data + 4 * dy.offset
        return self._take("layer_norm_bwd", [(x.data + 4 * x.offset, n), (src, n), (w, cols), (mean, n // cols), (rstd, n // cols)],
                          [(dx, n), (dw, cols), (db, cols), (work, 16)], src, dx, n)


class HostBackend:
    name, defers, ordinal = "host", False, 0

    def __init__(self):
        self.lib, self.handle = HostLib(), 1

    def close(self):
        self.handle = None

    def check(self, status):
        if status:
            raise BackendError(status, "refused")

    def alloc(self, n, dt):
        return DeviceStorage(self.lib.new(n, dt), self)

    def from_host(self, a):
        a = np.asarray(a)
        s = self.alloc(a.size, DType.of(a))
        self.lib.memory[s.handle][0][:a.size] = a.reshape(-1)
        return s

    def to_host(self, s, l, dt):
        return self.lib.memory[s.handle][0][l.offsets()]

    def copy_strided(self, src, ls, dt, dst, ld):
        self.lib.memory[dst.handle][0][ld.offsets()] = self.lib.memory[src.handle][0][ls.offsets()]

    def reduce(self, op, s, l, dt, axis):
        raise AssertionError("not used here")
