"""Layer norm, gradient norm and the many-tensor Adam at the edges of what their documentation allows, on the GPU."""
import ctypes

import numpy as np
import pytest

from weta_b200 import layers, optim
from weta_b200.backend import B200Backend, BackendError
from weta_b200.core import BinaryOp, DType, Layout
from weta_b200.fusion import FusingBackend

pytestmark = pytest.mark.gpu
F = np.float32
U = {DType.F32: 2.0 ** -24, DType.F64: 2.0 ** -53}
NP = {DType.F32: np.float32, DType.F64: np.float64}


def down(be, s, n, dt=DType.F32):
    return be.to_host(s, Layout.contiguous([n]), dt).copy()


@pytest.mark.parametrize("dropped", [False, True])
def test_a_deferred_gradient_assigned_to_a_storage_that_changes(gpu, dropped):
    """g is assigned to a buffer, which is overwritten between set_grads and the step: the step's result is the plain backend's."""
    n = 700
    l = Layout.contiguous([n])
    rng = np.random.default_rng(5)
    a, other, start = (rng.standard_normal(n).astype(F) for _ in range(3))
    results = []
    for be in (gpu, FusingBackend(gpu)):
        sa, so, theta, buf = (gpu.from_host(v) for v in (a, other, start, start))
        opt = optim.AdamMulti(be, [theta], lr=0.1)
        g = be.binary(BinaryOp.ADD, sa, l, sa, l, DType.F32)
        be.copy_strided(g, l, DType.F32, buf, l)
        opt.set_grads([g])
        if dropped:
            del g
        be.copy_strided(so, l, DType.F32, buf, l)
        norm, clip = opt.grad_norm(1.0)
        opt.step(1, clip)
        results.append((down(be, theta, n), down(be, norm, 1), down(be, buf, n)))
    for p, q in zip(*results):
        assert np.array_equal(p, q)
    assert np.array_equal(results[0][2], other)


BIG = {DType.F32: 1e36, DType.F64: 1e306}


@pytest.mark.parametrize("cols", [3, 21, 36, 64, 131, 200, 256, 257, 520, 777, 1024, 1544, 3080, 4100, 5001, 8192, 9000, 9001, 17000])
@pytest.mark.parametrize("dt", [DType.F32, DType.F64])
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_of_one_huge_value_have_a_finite_gradient(gpu, cols, dt, shift):
    """xhat is 0 in such a row however large the value, and dx = rstd (g - mean g); the statistics are given, since the forward
    pass's sum of that many such values may overflow.  The widths fill a thread's last vector and leave it partly empty.
    Tolerance as for every row: 60 u rstd (|g| + mean |g|), and u |xhat| terms that are 0 here."""
    rng = np.random.default_rng(cols + shift)
    rows, rstd = 5, 1024.0
    u, t = U[dt], NP[dt]
    x = rng.standard_normal((rows, cols)).astype(t)
    mean = x.mean(1).astype(t)
    for k, v in ((1, BIG[dt]), (3, -BIG[dt]), (4, 2.0)):
        x[k] = mean[k] = v
    dy, w = rng.standard_normal((rows, cols)).astype(t), rng.uniform(0.5, 1.5, cols).astype(t)
    l = Layout.contiguous([rows, cols])
    sg = gpu.from_host(np.concatenate([np.zeros(shift, t), dy.reshape(-1)]))
    out = layers.layer_norm_bwd(gpu, gpu.from_host(x.reshape(-1)), l, sg, Layout([rows, cols], [cols, 1], shift), dt, 1, gpu.from_host(w),
                                gpu.from_host(mean), gpu.from_host(np.full(rows, rstd, t)))
    dx, dw, db = (down(gpu, s, n, dt) for s, n in zip(out, (rows * cols, cols, cols)))
    g = dy.astype(np.longdouble) * w
    xh = (x.astype(np.longdouble) - mean.astype(np.longdouble)[:, None]) * rstd
    s, p = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    bound = 60 * u * rstd * (np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(xh) * np.abs(g * xh).mean(1, keepdims=True))
    assert (np.abs(dx.reshape(rows, cols) - rstd * (g - s - xh * p)) <= bound).all()
    assert (np.abs(dw - (dy * xh).sum(0)) <= (16 + rows) * u * np.abs(dy * xh).sum(0)).all()
    assert (np.abs(db - dy.sum(0, dtype=np.longdouble)) <= (16 + rows) * u * np.abs(dy).sum(0)).all()


@pytest.mark.parametrize("eps,lr,scale", [(2.0 ** 100, 2.0 ** 110, 2.0 ** -26), (2.0 ** 90, 2.0 ** 100, 2.0 ** -40), (2.0 ** 60, 2.0 ** 70, 2.0 ** -55),
                                          (2.0 ** 66, 2.0 ** 80, 1.0), (1e-8, 1.0, 2.0 ** 41), (1e-8, 1.0, 2.0 ** 58)])
def test_8_bit_step_with_quotients_near_and_below_the_normal_range(gpu, eps, lr, scale):
    """m / (root + eps) rounded once, subnormal or not: theta starts at 0, so its first value is that quotient times lr.  Gradients
    lie within a factor of 8, and beta2 near 1 makes 1 / sqrt(1 - beta2^t) as large as 2^13."""
    from test_gpu_adam_multi import Plain, same

    n, b2 = 256 * 64, 1 - 2.0 ** -26
    rng = np.random.default_rng(2)
    g = (rng.uniform(1, 8, n) * rng.choice([-1, 1], n) * scale).astype(F)
    th = np.zeros(n, F)
    store = gpu.from_host(th)
    opt = optim.AdamMulti(gpu, [store], 8, lr=lr, betas=(0.9, b2), eps=eps)
    opt.set_grads([gpu.from_host(g)])
    p = Plain(n, 8)
    with np.errstate(all="ignore"):
        for t in (1, 2):
            opt.step(t)
            th = p.step(th, g, t, lr, 0.9, b2, eps, 0.0, False, False, None)
            assert np.abs(th).max() > 0 and same(down(gpu, store, n), th), t


@pytest.mark.parametrize("c", [3, 5, 7, 11, 13])
def test_8_bit_step_with_subnormal_quotients_half_way_between_two(gpu, c):
    """With both betas 0 the first step is theta - g / (|g| + eps) lr, and |g| + eps rounds to eps = c 2^98.  g = c (2k + 1) 2^-52
    makes the quotient (2k + 1) 2^-150, half way between two subnormal values: it goes to the even one."""
    from test_gpu_adam_multi import Plain, same

    n, eps, lr = 256 * 64, c * 2.0 ** 98, 2.0 ** 120
    k = np.arange(8, n + 8)
    g = (c * (2 * k + 1) * 2.0 ** -52).astype(F)
    assert (g.astype(np.float64) == c * (2 * k + 1) * 2.0 ** -52).all()
    store = gpu.zeros(n, DType.F32)
    opt = optim.AdamMulti(gpu, [store], 8, lr=lr, betas=(0.0, 0.0), eps=eps)
    opt.set_grads([gpu.from_host(g)])
    opt.step(1)
    even = (k + (k & 1)) * 2.0 ** (120 - 149)
    got = down(gpu, store, n)
    assert np.array_equal(got, -even.astype(F))
    assert same(got, Plain(n, 8).step(np.zeros(n, F), g, 1, lr, 0.0, 0.0, eps, 0.0, False, False, None))


def norm_twice(be, n=512):
    """A forward and a backward call that both wait for copies; the sum of their outputs' bits."""
    rng = np.random.default_rng(n)
    l, x = Layout.contiguous([7, n]), be.from_host(rng.standard_normal(7 * n).astype(F))
    y, m, r = layers.layer_norm_fwd(be, x, l, DType.F32, 1)
    dx, _, _ = layers.layer_norm_bwd(be, x, l, y, l, DType.F32, 1, None, m, r)
    return down(be, y, 7 * n), down(be, dx, 7 * n)


def test_a_wait_that_runs_out_is_seen_by_its_own_backend_only(gpu):
    """The hook lets the kernels' bounded wait run out on one backend; another backend's check neither reports nor clears it,
    and both go on working.  A GEMM's flag that is up at the same time is cleared by the same check."""
    for f in (gpu.lib.wb_layer_norm_selftest_timeout, gpu.lib.wb_gemm_selftest_timeout):
        f.argtypes, f.restype = [ctypes.c_void_p, ctypes.c_int], ctypes.c_int
    be = B200Backend(0)
    fresh = B200Backend(0)
    before = norm_twice(be)
    gpu.gemm_check()
    be.gemm_check()
    be.check(be.lib.wb_layer_norm_selftest_timeout(be.handle, 64))
    be.synchronize()
    norm_twice(gpu)
    gpu.gemm_check()
    fresh.gemm_check()
    with pytest.raises(BackendError, match="layer norm gave up"):
        be.gemm_check()
    be.gemm_check()
    be.check(be.lib.wb_layer_norm_selftest_timeout(be.handle, 64))
    be.check(be.lib.wb_gemm_selftest_timeout(be.handle, 64))
    with pytest.raises(BackendError, match="gave up") as e:
        be.gemm_check()
    assert e.value.status == 6
    be.gemm_check()
    for a, b in zip(before, norm_twice(be)):
        assert np.array_equal(a, b)
    be.gemm_check()
    be.close()
    fresh.close()


def test_the_first_call_of_a_backend_may_be_captured(gpu):
    """Whatever a backend needs for its waits is made without disturbing a capture."""
    import torch

    rows, n = 7, 9000
    st = torch.cuda.Stream()
    be = B200Backend(0, stream=st.cuda_stream)
    t = {k: torch.zeros(s, device="cuda") for k, s in dict(x=(rows, n), y=(rows, n), m=(rows,), r=(rows,), dx=(rows, n)).items()}
    torch.cuda.synchronize()
    s = {k: be.wrap_pointer(a.data_ptr(), a.numel(), DType.F32) for k, a in t.items()}
    l = Layout.contiguous([rows, n])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        layers.layer_norm_fwd(be, s["x"], l, DType.F32, 1, out=(s["y"], s["m"], s["r"]))
        layers.layer_norm_bwd(be, s["x"], l, s["y"], l, DType.F32, 1, None, s["m"], s["r"], out=(s["dx"], None, None))
    rng = np.random.default_rng(n)
    x = rng.standard_normal((rows, n)).astype(F)
    t["x"].copy_(torch.from_numpy(x))
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        graph.replay()
    torch.cuda.synchronize()
    be.gemm_check()
    xs = gpu.from_host(x.reshape(-1))
    y, m, r = layers.layer_norm_fwd(gpu, xs, l, DType.F32, 1)
    dx, _, _ = layers.layer_norm_bwd(gpu, xs, l, y, l, DType.F32, 1, None, m, r)
    assert np.array_equal(t["y"].cpu().numpy().reshape(-1), down(gpu, y, rows * n))
    assert np.array_equal(t["dx"].cpu().numpy().reshape(-1), down(gpu, dx, rows * n))
    del graph
    s.clear()


ROWS = [(1, 1), (1, 1024), (2, 64), (3, 7), (5, 9001), (7, 96), (33, 1000), (128, 512), (297, 40), (1000, 33), (2500, 256), (4099, 100), (70001, 3), (3001, 777),
        (1201, 2048), (1111, 4100), (1400, 4096), (700, 8192), (601, 9000), (400, 9001), (330, 16388), (20011, 33), (9000, 250), (6007, 130),
        (4443, 1000), (2368, 12), (300, 20001), (90, 33000)]


@pytest.mark.parametrize("dt", [DType.F32, DType.F64])
@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("form", ["plain", "shifted", "strided"])
def test_each_row_counts_once_in_the_sums(gpu, rows, cols, dt, form):
    """Small whole numbers, mean 1 or 2, rstd 1: every partial sum of dweight and dbias is a whole number under 2^24 and exact in
    any order, and every row adds at least 1 to every column, so a row left out or taken twice shows in each."""
    if form == "strided" and rows * cols > 1 << 20:
        pytest.skip("the kernel for any view is covered by the smaller shapes")
    rng = np.random.default_rng(rows + cols)
    t = NP[dt]
    mean = rng.integers(1, 3, rows)
    x = mean[:, None] + rng.integers(1, 4, (rows, cols))
    dy = rng.integers(1, 3, (rows, cols))
    assert 6 * rows < 1 << 24
    dw, db = (dy * (x - mean[:, None])).sum(0), dy.sum(0)
    lx = lg = Layout.contiguous([rows, cols])
    xs, gs = x.astype(t).reshape(-1), dy.astype(t).reshape(-1)
    if form == "shifted":
        gs, lg = np.concatenate([np.zeros(1, t), gs]), Layout([rows, cols], [cols, 1], 1)
    if form == "strided":
        xs, lx = np.ascontiguousarray(x.astype(t).T).reshape(-1), Layout([rows, cols], [1, rows], 0)
    args = (gpu, gpu.from_host(xs), lx, gpu.from_host(gs), lg, dt, 1, None, gpu.from_host(mean.astype(t)), gpu.from_host(np.ones(rows, t)))
    for out in (None, (None, gpu.alloc(cols, dt), gpu.alloc(cols, dt))):
        _, w, b = layers.layer_norm_bwd(*args, out=out)
        assert np.array_equal(down(gpu, w, cols, dt), dw.astype(t)) and np.array_equal(down(gpu, b, cols, dt), db.astype(t))


@pytest.mark.parametrize("rows,cols", [s for s in ROWS if s[1] <= 8192])
def test_sums_over_rows_are_added_in_short_chains(gpu, rows, cols):
    """Rows of up to 8192 f32 columns.  A thread adds the terms of at most rows / 148 rows beyond one span of its block (32 rows),
    or of three spans where few blocks run; the block joins at most 64 threads per column in f32, the blocks at most eight in f32
    (a cluster) or all of them in f64, and a term is rounded three times itself: (rows / 148 + 96 + 64 + 8 + 4) u of the sum of
    magnitudes."""
    rng = np.random.default_rng(rows * 3 + cols)
    x, dy = (rng.standard_normal((rows, cols)).astype(F) for _ in range(2))
    mean, rstd = (rng.standard_normal(rows) * 0.1).astype(F), rng.uniform(0.5, 2, rows).astype(F)
    l = Layout.contiguous([rows, cols])
    _, dw, db = layers.layer_norm_bwd(gpu, gpu.from_host(x.reshape(-1)), l, gpu.from_host(dy.reshape(-1)), l, DType.F32, 1, None, gpu.from_host(mean),
                                      gpu.from_host(rstd))
    terms = dy.astype(np.float64) * ((x.astype(np.float64) - mean[:, None]) * rstd[:, None])
    chain = (rows / 148 + 172) * 2.0 ** -24
    assert (np.abs(down(gpu, dw, cols) - terms.sum(0)) <= chain * np.abs(terms).sum(0)).all()
    assert (np.abs(down(gpu, db, cols) - dy.sum(0, dtype=np.float64)) <= chain * np.abs(dy).sum(0, dtype=np.float64)).all()


def test_roots_reciprocals_and_quotients_of_the_8_bit_step_are_rounded(gpu):
    """Every root and reciprocal of the range that the step uses them in, and four billion quotients."""
    f = gpu.lib.wb_adam_multi_selftest_rounding
    f.argtypes, f.restype = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_int64)], ctypes.c_int
    wrong = (ctypes.c_int64 * 4)(-1, -1, -1, -1)
    gpu.check(f(gpu.handle, wrong))
    assert list(wrong) == [0, 0, 0, (180 + 121) * 2 ** 23 + 4]  # two at a time, both ends included
    assert f(None, wrong) == 1 and f(gpu.handle, None) == 1
