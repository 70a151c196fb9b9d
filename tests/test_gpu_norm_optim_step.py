"""Layer norm, gradient norm and many-tensor AdamW together, the way a training step uses them: linear -> layer norm ->
linear -> softmax cross-entropy, its backward pass, clipping, and the step over all six tensors, against 64 bits.

Contractions run in FP32 mode with inner lengths of at most 130, so each errs by at most 146 u (8.7e-6) of its largest
magnitude; the layer norm multiplies an error by at most rstd * max|weight| (under 3 here), and three contractions and two
layer-norm passes lie on the longest path: 1e-4 of a gradient's largest magnitude bounds them together."""
import ctypes
import math

import numpy as np
import pytest

from weta_b200 import layers, optim
from weta_b200.backend import BackendError
from weta_b200.core import BinaryOp, DType, Layout
from weta_b200.fusion import FusingBackend
from weta_b200.trainer import _declare

pytestmark = pytest.mark.gpu
N, IN, HID, OUT = 64, 96, 130, 10
U = 2.0 ** -24
LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.999, 1e-8, 0.1
SHAPES = [(HID, IN), (HID,), (HID,), (HID,), (OUT, HID), (OUT,)]  # w1, b1, gain, shift, w2, b2
NO_DECAY = [False, True, True, True, False, True]


def plain(params, x, y):
    """Gradients of the mean cross-entropy in f64."""
    w1, b1, g, s, w2, b2 = (p.astype(np.float64) for p in params)
    h = x @ w1.T + b1
    mu = h.mean(1, keepdims=True)
    r = 1 / np.sqrt(h.var(1, keepdims=True) + 1e-5)
    xh = (h - mu) * r
    z = xh * g + s
    o = z @ w2.T + b2
    p = np.exp(o - o.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    do = p.copy()
    do[np.arange(N), y] -= 1
    do /= N
    dz = do @ w2
    a = dz * g
    dh = r * (a - a.mean(1, keepdims=True) - xh * (a * xh).mean(1, keepdims=True))
    return [dh.T @ x, dh.sum(0), (dz * xh).sum(0), dz.sum(0), do.T @ z, do.sum(0)]


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(gpu, bits):
    _declare(gpu.lib)
    lib, H = gpu.lib, gpu.handle
    rng = np.random.default_rng(17)
    x, y = rng.standard_normal((N, IN)).astype(np.float32), rng.integers(0, OUT, N)
    params = [(rng.standard_normal(s) / math.sqrt(s[-1])).astype(np.float32) for s in SHAPES]
    params[2] = np.ones(HID, np.float32) + 0.1 * params[2]
    sizes = [p.size for p in params]
    ps = [gpu.from_host(p.reshape(-1)) for p in params]
    gs = [gpu.alloc(n, DType.F32) for n in sizes]
    xs, ys = gpu.from_host(x.reshape(-1)), gpu.from_host(y.astype(np.int64))
    h, z, dz, dh = (gpu.alloc(N * HID, DType.F32) for _ in range(4))
    o, do, loss = gpu.alloc(N * OUT, DType.F32), gpu.alloc(N * OUT, DType.F32), gpu.alloc(1, DType.F32)
    lay = Layout.contiguous([N, HID])
    get = lambda s, n: gpu.to_host(s, Layout.contiguous([n]), DType.F32)
    opt = optim.AdamMulti(gpu, ps, bits, NO_DECAY, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, decoupled=True)
    opt.set_grads(gs)
    moments = [(np.zeros(n), np.zeros(n)) for n in sizes]
    gpu.set_matmul_mode(2)
    try:
        for t in (1, 2, 3):
            now = [get(s, n) for s, n in zip(ps, sizes)]
            gpu.check(lib.wb_linear_fwd(H, xs.ptr, ps[0].ptr, ps[1].ptr, N, IN, HID, 0, h.ptr))
            _, mean, rstd = layers.layer_norm_fwd(gpu, h, lay, DType.F32, 1, ps[2], ps[3], 1e-5,
                                                  out=(z, gpu.alloc(N, DType.F32), gpu.alloc(N, DType.F32)))
            gpu.check(lib.wb_linear_fwd(H, z.ptr, ps[4].ptr, ps[5].ptr, N, HID, OUT, 0, o.ptr))
            gpu.check(lib.wb_softmax_ce(H, o.ptr, ys.ptr, N, OUT, None, do.ptr, None, loss.ptr, 1.0))
            gpu.check(lib.wb_linear_bwd(H, z.ptr, ps[4].ptr, do.ptr, N, HID, OUT, dz.ptr, gs[4].ptr, gs[5].ptr))
            layers.layer_norm_bwd(gpu, h, lay, dz, lay, DType.F32, 1, ps[2], mean, rstd, out=(dh, gs[2], gs[3]))
            gpu.check(lib.wb_linear_bwd(H, xs.ptr, ps[0].ptr, dh.ptr, N, IN, HID, None, gs[0].ptr, gs[1].ptr))
            norm, clip = opt.grad_norm(0.25)
            before = [get(s, opt.state_len).astype(np.float64) for s in opt.read_state()]
            opt.step(t, clip)

            got = [get(s, n).astype(np.float64) for s, n in zip(gs, sizes)]
            for a, b in zip(got, plain([p.reshape(s) for p, s in zip(now, SHAPES)], x.astype(np.float64), y)):
                assert np.abs(a - b.reshape(-1)).max() <= 1e-4 * np.abs(b).max()
            total = math.sqrt(sum((g * g).sum() for g in got))
            factor = min(1.0, 0.25 / (total + 1e-6))
            assert factor < 1 and abs(get(norm, 1)[0] - total) <= 2 * U * total and abs(get(clip, 1)[0] - factor) <= 2 * U * factor
            for k, n in enumerate(sizes):
                if bits == 32:
                    m, v = moments[k]
                else:  # the moments that the 8-bit state stood for
                    at = opt.offset(k)
                    m, v = (b[at:at + n] if t > 1 else np.zeros(n) for b in before)
                g = got[k] * factor
                m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
                moments[k] = (m, v)
                th = now[k].astype(np.float64) * (1 if NO_DECAY[k] else 1 - LR * WD)
                step = LR / (1 - B1 ** t) * m / (np.sqrt(v) / math.sqrt(1 - B2 ** t) + EPS)
                # the chain rounds at most 16 times on the way to the update, 3 times the weight, and m of a few steps may
                # cancel: its error is relative to |m| summed without signs, at most LR of update per step
                room = 3 * U * np.abs(th) + 64 * t * U * np.maximum(np.abs(step), LR)
                assert (np.abs(get(ps[k], n) - (th - step)) <= room).all(), (t, k)
    finally:
        gpu.set_matmul_mode(0)
    gpu.gemm_check()


def test_through_the_fusing_backend(gpu):
    """Pending operands are evaluated, what reads a storage is evaluated before it is written over, and a pending value is no output."""
    fb = FusingBackend(gpu)
    rng = np.random.default_rng(3)
    rows, cols = 6, 100
    l, lc, one = Layout.contiguous([rows, cols]), Layout.contiguous([cols]), Layout.contiguous([1])
    flat = Layout.contiguous([rows * cols])
    x, dy = (rng.standard_normal(rows * cols).astype(np.float32) for _ in range(2))
    w, b = (rng.standard_normal(cols).astype(np.float32) for _ in range(2))
    down = lambda s, n: fb.to_host(s, Layout.contiguous([n]), DType.F32).copy()
    keep = []

    def twice(a, lay):
        keep.append(gpu.from_host(a))
        return fb.binary(BinaryOp.ADD, keep[-1], lay, keep[-1], lay, DType.F32)

    want = layers.layer_norm_fwd(gpu, gpu.from_host(x + x), l, DType.F32, 1, gpu.from_host(w + w), gpu.from_host(b + b))
    got = layers.layer_norm_fwd(fb, twice(x, l), l, DType.F32, 1, twice(w, lc), twice(b, lc))
    for a, c, n in zip(got, want, (rows * cols, rows, rows)):
        assert np.array_equal(down(a, n), down(c, n))
    args = (l, DType.F32, 1)
    wanted = layers.layer_norm_bwd(gpu, gpu.from_host(x + x), l, gpu.from_host(dy + dy), *args, gpu.from_host(w + w), *want[1:])
    grads = layers.layer_norm_bwd(fb, twice(x, l), l, twice(dy, l), *args, twice(w, lc), *got[1:])
    for a, c, n in zip(grads, wanted, (rows * cols, cols, cols)):
        assert np.array_equal(down(a, n), down(c, n))

    y = got[0]
    old = down(y, rows * cols)
    pending = fb.binary(BinaryOp.ADD, y, flat, y, flat, DType.F32)
    layers.layer_norm_fwd(fb, gpu.from_host(dy), l, DType.F32, 1, out=got)
    assert np.array_equal(down(pending, rows * cols), old + old) and not np.array_equal(down(y, rows * cols), old)
    with pytest.raises(BackendError, match="can't be written over"):
        layers.layer_norm_fwd(fb, gpu.from_host(dy), l, DType.F32, 1, out=(twice(x, l), None, None))

    theta, other = gpu.from_host(x), gpu.from_host(x)
    lazy, plain_ = optim.AdamMulti(fb, [theta], lr=0.1), optim.AdamMulti(gpu, [other], lr=0.1)
    lazy.set_grads([twice(dy, flat)])
    plain_.set_grads([gpu.from_host(dy + dy)])
    pending = fb.binary(BinaryOp.ADD, theta, flat, theta, flat, DType.F32)
    half = np.full(1, 0.25, np.float32)
    lazy.step(1, twice(half, one))
    plain_.step(1, gpu.from_host(half + half))
    assert np.array_equal(down(pending, rows * cols), x + x)
    assert np.array_equal(down(theta, rows * cols), down(other, rows * cols))
    assert np.array_equal(down(lazy.grad_norm(1.0)[0], 1), down(plain_.grad_norm(1.0)[0], 1))
    assert np.array_equal(down(lazy.read_state()[1], lazy.state_len), down(plain_.read_state()[1], lazy.state_len))
    with pytest.raises(BackendError, match="can't be written over"):
        optim.AdamMulti(fb, [twice(x, flat)])
