"""Layer normalisation, forward and backward, against a plain implementation in 64 bits.

Tolerances, with u half a step of the type and A the row's mean magnitude.  A sum of n terms in a tree of chains errs by
at most (longest chain + depth) u times the sum of magnitudes; no kernel chains more than 48 additions and levels along a
row (the kernel for any view sums in f64).  So the mean errs by 48 u A, a deviation by that plus u of itself, and the
relative error of rstd is at most 48 u + 0.5 (48 u A rstd)^2 + 4 u.  `FWD` and `BWD` below add these up per element.
A column of the weight's gradient is a sum over the rows: (16 + rows) u times the sum of magnitudes bounds any order.
"""
import ctypes

import numpy as np
import pytest

from weta_b200 import layers
from weta_b200.core import DType, Layout

pytestmark = pytest.mark.gpu

U = {DType.F32: 2.0 ** -24, DType.F64: 2.0 ** -53}
NP = {DType.F32: np.float32, DType.F64: np.float64}


def values(rng, shape, dt, offset=0.5):
    x = rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[:-1] + (1,))) + offset * rng.standard_normal(shape[:-1] + (1,))
    return x.astype(NP[dt])


def plain_fwd(x, w, b, eps):
    """[rows, cols] in longdouble: mean, rstd, y, and the bound on y's and rstd's error in units of u."""
    x = x.astype(np.longdouble)
    mean = x.mean(1, keepdims=True)
    d = x - mean
    rstd = 1 / np.sqrt((d * d).mean(1, keepdims=True) + np.longdouble(eps))
    xh = d * rstd
    y = xh * (1 if w is None else w) + (0 if b is None else b)
    return mean[:, 0], rstd[:, 0], xh, y


def check_fwd(x, w, b, eps, dt, y, mean, rstd):
    u = U[dt]
    m0, r0, xh, y0 = plain_fwd(x, w, b, eps)
    a = np.abs(x).mean(1).astype(np.longdouble)
    rel = 52 * u + 0.5 * (48 * u * a * r0) ** 2
    assert (np.abs(mean - m0) <= 49 * u * a).all()
    assert (np.abs(rstd - r0) <= rel * r0).all()
    wide = 1.0 if w is None else np.abs(w).astype(np.longdouble)
    bound = wide * (49 * u * (a * r0)[:, None] + (rel[:, None] + 4 * u) * np.abs(xh)) + 2 * u * np.abs(y0)
    assert (np.abs(y - y0) <= bound).all(), float((np.abs(y - y0) / np.maximum(bound, 1e-300)).max())


def check_bwd(x, dy, w, mean, rstd, dt, dx, dw, db):
    u = U[dt]
    x, dy = x.astype(np.longdouble), dy.astype(np.longdouble)
    rs, n = rstd.astype(np.longdouble)[:, None], x.shape[1]
    xh = (x - mean.astype(np.longdouble)[:, None]) * rs
    g = dy * (1 if w is None else w.astype(np.longdouble))
    s, p = g.sum(1, keepdims=True) / n, (g * xh).sum(1, keepdims=True) / n
    if dx is not None:
        # s errs by 50 u mean|g|, p by 54 u mean|g xh|, and each of the three terms by 4 u of itself
        bound = 60 * u * np.abs(rs) * (np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(xh) * np.abs(g * xh).mean(1, keepdims=True))
        d0 = rs * (g - s - xh * p)
        assert (np.abs(dx - d0) <= bound).all(), float((np.abs(dx - d0) / np.maximum(bound, 1e-300)).max())
    if dw is not None:
        assert (np.abs(dw - (dy * xh).sum(0)) <= (16 + x.shape[0]) * u * np.abs(dy * xh).sum(0)).all()
    if db is not None:
        assert (np.abs(db - dy.sum(0)) <= (16 + x.shape[0]) * u * np.abs(dy).sum(0)).all()


def get(gpu, s, shape, dt):
    return gpu.to_host(s, Layout.contiguous([int(np.prod(shape, dtype=np.int64))]), dt).reshape(shape)


def both_ways(gpu, rows, cols, dt, seed=0, affine=True, eps=1e-5, x=None, offset=0.5):
    rng = np.random.default_rng(seed + 31 * rows + cols)
    x = values(rng, (rows, cols), dt, offset) if x is None else x
    dy = values(rng, (rows, cols), dt)
    w, b = ((1 + 0.3 * rng.standard_normal(cols)).astype(NP[dt]), rng.standard_normal(cols).astype(NP[dt])) if affine else (None, None)
    l = Layout.contiguous([rows, cols])
    xs, gs = gpu.from_host(x.reshape(-1)), gpu.from_host(dy.reshape(-1))
    ws, bs = (gpu.from_host(w), gpu.from_host(b)) if affine else (None, None)
    ys, ms, rs = layers.layer_norm_fwd(gpu, xs, l, dt, 1, ws, bs, eps)
    mean, rstd = get(gpu, ms, (rows,), dt), get(gpu, rs, (rows,), dt)
    check_fwd(x, w, b, eps, dt, get(gpu, ys, (rows, cols), dt), mean, rstd)
    dxs, dws, dbs = layers.layer_norm_bwd(gpu, xs, l, gs, l, dt, 1, ws, ms, rs)
    check_bwd(x, dy, w, mean, rstd, dt, get(gpu, dxs, (rows, cols), dt), get(gpu, dws, (cols,), dt), get(gpu, dbs, (cols,), dt))


COLS = [1, 2, 3, 4, 5, 8, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 384, 500, 512, 513, 777, 1000, 1001, 1023, 1024, 1025, 1500,
        2000, 2047, 2048, 2049, 4000, 4096, 4097, 5001, 8000, 8192, 8193, 10000, 12289, 16384, 16385, 20000, 32768, 40001]


@pytest.mark.parametrize("dt", [DType.F32, DType.F64])
@pytest.mark.parametrize("cols", COLS)
def test_columns(gpu, cols, dt):
    both_ways(gpu, 5, cols, dt)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 1024), (2, 64), (7, 96), (33, 1000), (128, 512), (297, 40), (1000, 33), (2500, 256), (4099, 100),
                                       (70001, 3), (3001, 777), (1201, 2048), (1111, 4100), (1400, 4096), (700, 8192), (601, 9000), (400, 9001),
                                       (330, 16388), (20011, 33), (9000, 250), (6007, 130)])
def test_rows(gpu, rows, cols):
    both_ways(gpu, rows, cols, DType.F32)


@pytest.mark.parametrize("rows,cols", [(3000, 65), (2500, 129), (1500, 1000), (801, 2049), (500, 4099), (310, 6000)])
def test_rows_in_double_precision(gpu, rows, cols):
    both_ways(gpu, rows, cols, DType.F64)


@pytest.mark.parametrize("cols", [6, 256, 1001, 4096, 16384, 33000])
def test_without_weight_and_bias(gpu, cols):
    both_ways(gpu, 17, cols, DType.F32, affine=False)


@pytest.mark.parametrize("cols", [8, 250, 1024, 4096, 9001, 16384])
def test_rows_far_from_zero(gpu, cols):
    """Rows whose mean is up to hundreds of times their spread: the variance is taken from deviations."""
    both_ways(gpu, 9, cols, DType.F32, offset=300.0)


@pytest.mark.parametrize("dt", [DType.F32, DType.F64])
@pytest.mark.parametrize("cols", [1, 7, 256, 1024, 4100, 20000])
def test_rows_of_one_value(gpu, cols, dt):
    """No spread: xhat is 0 (the mean of equal values is exact for powers of two), y the bias, rstd 1 / sqrt(eps)."""
    x = np.full((4, cols), 2.0, NP[dt])
    x[1] = -8.0
    l = Layout.contiguous([4, cols])
    b = np.arange(cols).astype(NP[dt])
    y, m, r = layers.layer_norm_fwd(gpu, gpu.from_host(x.reshape(-1)), l, dt, 1, None, gpu.from_host(b), 2.0 ** -16)
    assert np.array_equal(get(gpu, m, (4,), dt), x[:, 0])
    assert np.allclose(get(gpu, r, (4,), dt), 256.0, rtol=4 * U[dt], atol=0)
    assert np.array_equal(get(gpu, y, (4, cols), dt), np.broadcast_to(b, (4, cols)))


@pytest.mark.parametrize("cols", [3, 41, 97, 250, 1001, 3333, 9001, 12000, 20001])
def test_rows_of_one_integer(gpu, cols):
    """Sums of equal small integers are exact in any order, so the mean is that integer and y the bias, whatever 1 / cols is."""
    x = np.repeat(np.array([7.0, 200.0, -3.0], np.float32)[:, None], cols, 1)
    l = Layout.contiguous([3, cols])
    b = np.arange(cols).astype(np.float32)
    y, m, _ = layers.layer_norm_fwd(gpu, gpu.from_host(x.reshape(-1)), l, DType.F32, 1, None, gpu.from_host(b), 1e-12)
    assert np.array_equal(get(gpu, m, (3,), DType.F32), x[:, 0])
    assert np.array_equal(get(gpu, y, (3, cols), DType.F32), np.broadcast_to(b, (3, cols)))


@pytest.mark.parametrize("cols", [5, 300, 1024, 4096, 9001])
def test_values_that_are_not_finite_stay_in_their_row(gpu, cols):
    rng = np.random.default_rng(cols)
    x = values(rng, (6, cols), DType.F32)
    x[1, cols // 2], x[3, -1], x[4, 0] = np.nan, np.inf, -np.inf
    l = Layout.contiguous([6, cols])
    y, m, r = layers.layer_norm_fwd(gpu, gpu.from_host(x.reshape(-1)), l, DType.F32, 1, None, None, 1e-5)
    y = get(gpu, y, (6, cols), DType.F32)
    bad = [1, 3, 4]
    assert np.isnan(y[bad]).all()
    good = [0, 2, 5]
    check_fwd(x[good], None, None, 1e-5, DType.F32, y[good], get(gpu, m, (6,), DType.F32)[good], get(gpu, r, (6,), DType.F32)[good])
    dx, _, _ = layers.layer_norm_bwd(gpu, gpu.from_host(x.reshape(-1)), l, gpu.from_host(x.reshape(-1)), l, DType.F32, 1, None, m, r)
    dx = get(gpu, dx, (6, cols), DType.F32)
    assert np.isnan(dx[bad]).all() and np.isfinite(dx[good]).all()


def kind(a):
    """0 finite, 1 and -1 the infinities, 2 NaN."""
    return np.where(np.isnan(a), 2, np.where(np.isinf(a), np.sign(a), 0))


@pytest.mark.parametrize("cols", [21, 36, 40, 131, 200, 520, 777, 1544, 3080, 5001, 9000, 9001, 17000])
@pytest.mark.parametrize("dt", [DType.F32, DType.F64])
@pytest.mark.parametrize("shift", [0, 1])
def test_an_infinite_gradient_reaches_what_the_formula_says(gpu, cols, dt, shift):
    """An infinity in dy makes the row's dx infinite or NaN by the signs in the formula, and nothing else: a thread's places
    behind the row's end add nothing, not zero times the infinity.  `shift`: dy starts an element behind x's alignment."""
    rng = np.random.default_rng(cols + shift)
    rows = 6
    x, dy = (rng.standard_normal((rows, cols)).astype(NP[dt]) for _ in range(2))
    dy[1, 0], dy[2, cols - 1], dy[4, cols // 2] = np.inf, -np.inf, np.inf
    w = rng.uniform(0.5, 1.5, cols).astype(NP[dt])
    l = Layout.contiguous([rows, cols])
    sx, sw = gpu.from_host(x.reshape(-1)), gpu.from_host(w)
    sg = gpu.from_host(np.concatenate([np.zeros(shift, NP[dt]), dy.reshape(-1)]))
    _, mean, rstd = layers.layer_norm_fwd(gpu, sx, l, dt, 1, sw)
    dx, dw, db = layers.layer_norm_bwd(gpu, sx, l, sg, Layout([rows, cols], [cols, 1], shift), dt, 1, sw, mean, rstd)
    got = [get(gpu, a, b, dt) for a, b in ((dx, (rows, cols)), (dw, (cols,)), (db, (cols,)))]
    m, r = (get(gpu, a, (rows, 1), dt).astype(np.longdouble) for a in (mean, rstd))
    with np.errstate(invalid="ignore"):
        xh = (x.astype(np.longdouble) - m) * r
        g = dy.astype(np.longdouble) * w
        want = (r * (g - g.sum(1, keepdims=True) - xh * (g * xh).sum(1, keepdims=True)), (dy * xh).sum(0), dy.astype(np.longdouble).sum(0))
    for a, b in zip(got, want):
        assert np.array_equal(kind(a), kind(b))


VIEWS = {  # name: (storage length, Layout, normalised dims)
    "two normalised dims": (5 * 6 * 7, Layout.contiguous([5, 6, 7]), 2),
    "all dims": (6 * 7, Layout.contiguous([6, 7]), 2),
    "one dim": (300, Layout.contiguous([300]), 1),
    "slice of wider rows": (9 * 1040, Layout([9, 1000], [1040, 1], 8), 1),
    "slice at an odd offset": (9 * 1040, Layout([9, 1000], [1040, 1], 3), 1),
    "slice of odd rows": (9 * 517 + 5, Layout([9, 512], [517, 1], 1), 1),
    "transposed": (40 * 65, Layout([65, 40], [1, 65], 0), 1),
    "permuted outer dims": (4 * 5 * 96, Layout([5, 4, 96], [96, 480, 1], 0), 1),
    "permuted with a gap": (4 * 6 * 128, Layout([5, 4, 128], [128, 768, 1], 0), 1),
    "rows back to front": (7 * 64, Layout([7, 64], [-64, 1], 6 * 64), 1),
    "columns back to front": (7 * 64, Layout([7, 64], [64, -1], 63), 1),
    "every other column": (7 * 200, Layout([7, 100], [200, 2], 1), 1),
    "one row for all": (256, Layout([11, 256], [0, 1], 0), 1),
    "one value per row": (11, Layout([11, 64], [1, 0], 0), 1),
    "broadcast middle": (3 * 32, Layout([3, 4, 32], [32, 0, 1], 0), 1),
    "inner dims that do not merge": (3 * 8 * 16, Layout([3, 16, 8], [128, 1, 16], 0), 2),
    "slice of short odd rows": (50 * 101 + 9, Layout([50, 100], [101, 1], 1), 1),
    "slice of wide rows": (7 * 9100, Layout([7, 9001], [9100, 1], 2), 1),
    "slice of wider odd rows": (3 * 20011 + 5, Layout([3, 20000], [20011, 1], 5), 1),
    "wide rows back to front": (4 * 12000, Layout([4, 12000], [-12000, 1], 3 * 12000), 1),
    "a wide row for all": (10004, Layout([9, 10000], [0, 1], 3), 1),
    "more columns than a cluster holds": (2 * 70000, Layout.contiguous([2, 70000]), 1),
    "eight dims": (2 ** 6 * 9, Layout.contiguous([2, 1, 2, 2, 1, 2, 4, 9]), 3),
}


@pytest.mark.parametrize("dt", [DType.F32, DType.F64])
@pytest.mark.parametrize("name", list(VIEWS))
def test_views(gpu, name, dt):
    """x strided with dy contiguous, and the other way round."""
    length, l, nd = VIEWS[name]
    rng = np.random.default_rng(len(name))
    store = (rng.standard_normal(length) + 0.2).astype(NP[dt])
    x = store[l.offsets()]
    rows, cols = l.rows_cols(nd)
    x = x.reshape(rows, cols)
    dense = Layout.contiguous(l.shape)
    other = rng.standard_normal((rows, cols)).astype(NP[dt])
    w, b = rng.standard_normal(cols).astype(NP[dt]), rng.standard_normal(cols).astype(NP[dt])
    ss, os_, ws, bs = (gpu.from_host(a.reshape(-1)) for a in (store, other, w, b))
    y, m, r = layers.layer_norm_fwd(gpu, ss, l, dt, nd, ws, bs, 1e-3)
    mean, rstd = get(gpu, m, (rows,), dt), get(gpu, r, (rows,), dt)
    check_fwd(x, w, b, 1e-3, dt, get(gpu, y, (rows, cols), dt), mean, rstd)
    out = layers.layer_norm_bwd(gpu, ss, l, os_, dense, dt, nd, ws, m, r)
    check_bwd(x, other, w, mean, rstd, dt, *(get(gpu, s, sh, dt) for s, sh in zip(out, [(rows, cols), (cols,), (cols,)])))
    y, m, r = layers.layer_norm_fwd(gpu, os_, dense, dt, nd, ws, None, 1e-3)
    mean, rstd = get(gpu, m, (rows,), dt), get(gpu, r, (rows,), dt)
    out = layers.layer_norm_bwd(gpu, os_, dense, ss, l, dt, nd, ws, m, r)
    check_bwd(other, x, w, mean, rstd, dt, *(get(gpu, s, sh, dt) for s, sh in zip(out, [(rows, cols), (cols,), (cols,)])))


@pytest.mark.parametrize("dt", [DType.F32, DType.F64])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("rows,cols", [(3, 5), (9, 256), (5, 1001), (3, 4096), (2, 9000)])
def test_nothing_is_written_around_the_outputs(gpu, rows, cols, shift, dt):
    """Outputs (and inputs) at an offset of `shift` elements inside guarded buffers."""
    rng = np.random.default_rng(rows + cols)
    size, guard = DType.size(dt), 64
    bufs = {}

    def inside(n, data=None):
        a = np.full(n + 2 * guard, -7.0, NP[dt])
        if data is not None:
            a[guard + shift:guard + shift + n] = data.reshape(-1)
        s = gpu.from_host(a)
        bufs[s] = n
        return gpu.wrap_pointer(s.ptr + size * (guard + shift), n, dt)

    x, dy, w, b = (rng.standard_normal(s).astype(NP[dt]) for s in ((rows, cols), (rows, cols), (cols,), (cols,)))
    xs, gs, ws, bs = (inside(a.size, a) for a in (x, dy, w, b))
    ys, ms, rs, dxs, dws, dbs = (inside(n) for n in (rows * cols, rows, rows, rows * cols, cols, cols))
    need = gpu.lib.wb_layer_norm_bwd_workspace(gpu.handle, rows, cols, dt)
    room = gpu.from_host(np.full(need // size + 64, -7.0, NP[dt]))
    work = gpu.wrap_pointer(room.ptr, need // size, dt)
    l = Layout.contiguous([rows, cols])
    layers.layer_norm_fwd(gpu, xs, l, dt, 1, ws, bs, 1e-5, out=(ys, ms, rs))
    layers.layer_norm_bwd(gpu, xs, l, gs, l, dt, 1, ws, ms, rs, out=(dxs, dws, dbs), workspace=work)
    mean, rstd = get(gpu, ms, (rows,), dt), get(gpu, rs, (rows,), dt)
    check_fwd(x, w, b, 1e-5, dt, get(gpu, ys, (rows, cols), dt), mean, rstd)
    check_bwd(x, dy, w, mean, rstd, dt, get(gpu, dxs, (rows, cols), dt), get(gpu, dws, (cols,), dt), get(gpu, dbs, (cols,), dt))
    for s, n in bufs.items():
        a = get(gpu, s, (n + 2 * guard,), dt)
        assert (a[:guard + shift] == -7.0).all() and (a[guard + shift + n:] == -7.0).all()
    assert (get(gpu, room, (need // size + 64,), dt)[need // size:] == -7.0).all()


@pytest.mark.parametrize("cols", [48, 1000, 5000])
def test_single_gradients_equal_those_of_the_whole_call(gpu, cols):
    rng = np.random.default_rng(cols)
    rows, dt, l = 130, DType.F32, Layout.contiguous([130, cols])
    xs, gs, ws = (gpu.from_host(rng.standard_normal(n).astype(np.float32)) for n in (rows * cols, rows * cols, cols))
    _, m, r = layers.layer_norm_fwd(gpu, xs, l, dt, 1)
    whole = layers.layer_norm_bwd(gpu, xs, l, gs, l, dt, 1, ws, m, r)
    sizes = [rows * cols, cols, cols]
    for mask in range(8):
        out = [gpu.zeros(n, dt) if mask >> k & 1 else None for k, n in enumerate(sizes)]
        layers.layer_norm_bwd(gpu, xs, l, gs, l, dt, 1, ws, m, r, out=out)
        for k, n in enumerate(sizes):
            if out[k] is not None:
                assert np.array_equal(get(gpu, out[k], (n,), dt), get(gpu, whole[k], (n,), dt)), (mask, k)


def test_statistics_may_be_left_out_and_runs_repeat(gpu):
    rng = np.random.default_rng(1)
    l, dt = Layout.contiguous([700, 900]), DType.F32
    xs = gpu.from_host(rng.standard_normal(700 * 900).astype(np.float32))
    y0, m, r = layers.layer_norm_fwd(gpu, xs, l, dt, 1)
    for out in ((gpu.alloc(700 * 900, dt), None, None), (gpu.alloc(700 * 900, dt), m, None)):
        y, _, _ = layers.layer_norm_fwd(gpu, xs, l, dt, 1, out=out)
        assert np.array_equal(get(gpu, y, (630000,), dt), get(gpu, y0, (630000,), dt))
    first = layers.layer_norm_bwd(gpu, xs, l, y0, l, dt, 1, None, m, r)
    for _ in range(3):
        again = layers.layer_norm_bwd(gpu, xs, l, y0, l, dt, 1, None, m, r)
        for a, b, n in zip(first, again, (630000, 900, 900)):
            assert np.array_equal(get(gpu, a, (n,), dt), get(gpu, b, (n,), dt))


def test_no_rows(gpu):
    dt, l = DType.F32, Layout.contiguous([0, 12])
    x = gpu.alloc(0, dt)
    y, m, r = layers.layer_norm_fwd(gpu, x, l, dt, 1)
    dw, db = gpu.from_host(np.ones(12, np.float32)), gpu.from_host(np.ones(12, np.float32))
    layers.layer_norm_bwd(gpu, x, l, y, l, dt, 1, None, m, r, out=(None, dw, db))
    assert not get(gpu, dw, (12,), dt).any() and not get(gpu, db, (12,), dt).any()


def test_python_refusals_name_the_reason(gpu):
    from weta_b200.backend import BackendError

    x = gpu.zeros(32, DType.F32)
    with pytest.raises(BackendError, match="can't normalise the last 3 of 2 dims"):
        layers.layer_norm_fwd(gpu, x, Layout.contiguous([4, 8]), DType.F32, 3)
    with pytest.raises(BackendError, match="not a float"):
        layers.layer_norm_fwd(gpu, gpu.zeros(32, DType.I64), Layout.contiguous([4, 8]), DType.I64, 1)
    with pytest.raises(BackendError, match="overlaps"):
        layers.layer_norm_fwd(gpu, x, Layout.contiguous([4, 8]), DType.F32, 1, out=(x, None, None))
    with pytest.raises(BackendError, match="workspace holds 8 bytes"):
        m = gpu.zeros(4, DType.F32)
        layers.layer_norm_bwd(gpu, x, Layout.contiguous([4, 8]), gpu.zeros(32, DType.F32), Layout.contiguous([4, 8]), DType.F32, 1, None, m,
                              m, workspace=gpu.alloc(2, DType.F32))
    with pytest.raises(BackendError):
        layers.layer_norm_workspace(gpu, 4, 0, DType.F32)


@pytest.mark.parametrize("cols", [6, 40])
def test_gradients_against_differences(gpu, cols):
    """Central differences of sum(y * dy) in f64: with step h the quotient is off by O(h^2) and by u |loss| / h; at h = 1e-5
    and values near 1 both are under 1e-8 of the gradient's scale."""
    rng = np.random.default_rng(cols)
    rows, dt, h = 4, DType.F64, 1e-5
    l = Layout.contiguous([rows, cols])
    x, dy, w, b = (rng.standard_normal(s) for s in ((rows, cols), (rows, cols), (cols,), (cols,)))

    def loss(x, w, b):
        y, _, _ = layers.layer_norm_fwd(gpu, gpu.from_host(x.reshape(-1)), l, dt, 1, gpu.from_host(w), gpu.from_host(b), 1e-5)
        return float((get(gpu, y, (rows, cols), dt) * dy).sum())

    xs, ws = gpu.from_host(x.reshape(-1)), gpu.from_host(w)
    _, m, r = layers.layer_norm_fwd(gpu, xs, l, dt, 1, ws, None, 1e-5)
    grads = layers.layer_norm_bwd(gpu, xs, l, gpu.from_host(dy.reshape(-1)), l, dt, 1, ws, m, r)
    for which, (arr, g) in enumerate(zip((x, w, b), grads)):
        g = get(gpu, g, arr.shape, dt)
        for _ in range(12):
            at = tuple(rng.integers(0, n) for n in arr.shape)
            ends = []
            for sign in (1, -1):
                moved = [x.copy(), w.copy(), b.copy()]
                moved[which][at] += sign * h
                ends.append(loss(*moved))
            assert abs((ends[0] - ends[1]) / (2 * h) - g[at]) <= 1e-7 * max(1.0, abs(g[at]))


def test_large_offsets(gpu):
    """Rows that lie further than 2^31 elements from the view's start."""
    import torch

    rows, cols = 3, 1000
    big = torch.zeros(2 ** 31 + 2 ** 28, device="cuda")
    stride = 2 ** 30 + 12345
    x = torch.randn(rows, cols, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    for k in range(rows):
        big[k * stride:k * stride + cols] = x[k]
    torch.cuda.synchronize()
    xs = gpu.wrap_pointer(big.data_ptr(), big.numel(), DType.F32)
    l = Layout([rows, cols], [stride, 1])
    y, m, r = layers.layer_norm_fwd(gpu, xs, l, DType.F32, 1)
    mean, rstd = get(gpu, m, (rows,), DType.F32), get(gpu, r, (rows,), DType.F32)
    xn = x.cpu().numpy()
    check_fwd(xn, None, None, 1e-5, DType.F32, get(gpu, y, (rows, cols), DType.F32), mean, rstd)
    out = layers.layer_norm_bwd(gpu, xs, l, y, Layout.contiguous([rows, cols]), DType.F32, 1, None, m, r)
    check_bwd(xn, get(gpu, y, (rows, cols), DType.F32), None, mean, rstd, DType.F32,
              *(get(gpu, s, sh, DType.F32) for s, sh in zip(out, [(rows, cols), (cols,), (cols,)])))
    del big


def test_captured_on_another_stream(gpu):
    """Forward and backward captured twice, each graph with a workspace of its own, replayed side by side on new inputs."""
    import torch

    from weta_b200.backend import B200Backend

    rows, cols, dt = 600, 1024, DType.F32
    l = Layout.contiguous([rows, cols])
    runs = []
    for k in range(2):
        st = torch.cuda.Stream()
        be = B200Backend(0, stream=st.cuda_stream)
        t = {n: torch.zeros(sh, device="cuda") for n, sh in dict(x=(rows, cols), g=(rows, cols), y=(rows, cols), m=(rows,), r=(rows,),
                                                                 dx=(rows, cols), dw=(cols,), db=(cols,)).items()}
        torch.cuda.synchronize()
        s = {n: be.wrap_pointer(a.data_ptr(), a.numel(), dt) for n, a in t.items()}
        work = layers.layer_norm_workspace(be, rows, cols, dt)

        def call():
            layers.layer_norm_fwd(be, s["x"], l, dt, 1, out=(s["y"], s["m"], s["r"]))
            layers.layer_norm_bwd(be, s["x"], l, s["g"], l, dt, 1, None, s["m"], s["r"], out=(s["dx"], s["dw"], s["db"]), workspace=work)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call()
        runs.append((st, be, t, s, work, graph))
    gen = torch.Generator("cuda").manual_seed(9)
    for _ in range(3):
        for st, _, t, _, _, graph in runs:
            t["x"].normal_(generator=gen)
            t["g"].normal_(generator=gen)
        torch.cuda.synchronize()
        for st, _, _, _, _, graph in runs:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, t, _, _, _ in runs:
            a = {n: v.cpu().numpy() for n, v in t.items()}
            check_fwd(a["x"], None, None, 1e-5, dt, a["y"], a["m"], a["r"])
            check_bwd(a["x"], a["g"], None, a["m"], a["r"], dt, a["dx"], a["dw"], a["db"])
    for _, be, _, s, work, graph in runs:
        del graph
        s.clear()
    runs.clear()


def test_launch_counts_and_profile_label(gpu):
    l, dt = Layout.contiguous([64, 256]), DType.F32
    x = gpu.zeros(64 * 256, dt)
    out = (gpu.alloc(64 * 256, dt), None, None)
    before = gpu.launch_count()
    layers.layer_norm_fwd(gpu, x, l, dt, 1, out=out)
    assert gpu.launch_count() == before + 1
    gpu.set_profiling(True)
    try:
        layers.layer_norm_fwd(gpu, x, l, dt, 1, out=out)
    finally:
        gpu.set_profiling(False)
    assert "layer_norm" in gpu.profile_report()
