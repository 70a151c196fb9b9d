"""The many-tensor Adam step and gradient norm: bit for bit against a plain statement in f32 (every rounding is defined), against
wb_adam_step, and against 64 bits."""
import ctypes
import math

import numpy as np
import pytest

from weta_b200 import optim
from weta_b200.backend import BackendError
from weta_b200.core import DType, Layout
from weta_b200.trainer import _declare

pytestmark = pytest.mark.gpu
F = np.float32
U = 2.0 ** -24


def pad(n):
    return -(-n // 256) * 256


def down(gpu, s, n):
    return gpu.to_host(s, Layout.contiguous([n]), DType.F32)


class Plain:
    """One tensor's state and step, with each f32 operation rounded by itself."""

    def __init__(self, n, bits):
        self.n, self.bits, self.p = n, bits, pad(n)
        self.m, self.v = np.zeros(self.p, F), np.zeros(self.p, F)
        if bits == 8:
            self.mc, self.vc = np.zeros(self.p, np.int8), np.zeros(self.p, np.uint8)
            self.ms, self.vs = np.zeros(self.p // 256, F), np.zeros(self.p // 256, F)

    def read(self):
        if self.bits == 32:
            return self.m, self.v
        c = self.mc.astype(np.int32)
        with np.errstate(invalid="ignore"):
            m = (c * np.abs(c)).astype(F) * np.repeat(self.ms * F(1 / 16129), 256)
            c = self.vc.astype(np.int32)
            r = (c * c).astype(F) * np.repeat(self.vs * F(1 / 65025), 256)
            return m, r * r

    def step(self, theta, g, t, lr, b1, b2, eps, wd, decoupled, no_decay, scale):
        """The new theta; `scale` is None or the factor on the gradient."""
        n = self.n
        if scale is not None:
            g = g * F(scale)
        if wd and not no_decay:
            if decoupled:
                theta = theta * F(1 - lr * wd)
            else:
                g = g + theta * F(wd)
        m, v = (a[:n] for a in self.read())
        gm, gv = g * F(1 - b1), (g * g) * F(1 - b2)
        m, v = (gm, gv) if t == 1 else (m * F(b1) + gm, v * F(b2) + gv)
        root = np.sqrt(v)
        den = root * F(1 / math.sqrt(1 - power(b2, t))) + F(eps)
        with np.errstate(all="ignore"):
            theta = theta - (m / den) * F(lr / (1 - power(b1, t)))
        if self.bits == 32:
            self.m[:n], self.v[:n] = m, v
        else:
            self.encode(np.pad(m, (0, self.p - n)), np.pad(root, (0, self.p - n)))
        return theta

    def encode(self, m, root):
        for values, top, codes, scales in ((m, 127, "mc", "ms"), (root, 255, "vc", "vs")):
            a = np.abs(values).reshape(-1, 256)
            s = np.maximum(a.max(1), F(2.0 ** -100))
            bad = ~np.isfinite(s)
            s[bad] = F(1)
            with np.errstate(all="ignore"):
                c = np.minimum(np.rint(np.sqrt(np.where(bad[:, None], F(0), a) * (F(top * top) / s)[:, None])), F(top))
            if top == 255:
                c = np.where((a > 0) & (c < 1), F(1), c)
            c = np.where(values.reshape(-1, 256) < 0, -c, c).reshape(-1)
            self.__dict__[codes] = c.astype(np.int8 if top == 127 else np.uint8)
            self.__dict__[scales] = np.where(bad, F(np.nan), s)


def power(a, n):
    """Repeated squaring in f64, as the optimizer's scalars are made."""
    r = 1.0
    while True:
        if n & 1:
            r *= a
        n //= 2
        if n == 0:
            return r
        a *= a


def grads_for(rng, lens, spread=1.0):
    return [(0.01 * rng.standard_normal(n) * np.exp(spread * rng.standard_normal(n))).astype(F) for n in lens]


def state_of(gpu, opt, lens, bits):
    """The handle's state as lists per tensor, from the bytes."""
    p = opt.state_len
    raw = down(gpu, opt.state, opt.state_bytes // 4).view(np.uint8)
    out = []
    for i, n in enumerate(lens):
        o, q = opt.offset(i), pad(n)
        if bits == 32:
            f = raw.view(F)
            out.append((f[o:o + n], f[p + o:p + o + n]))
        else:
            sc = raw[2 * p:].view(F)
            out.append((raw[o:o + q].view(np.int8), raw[p + o:p + o + q], sc[o // 256:(o + q) // 256],
                        sc[p // 256 + o // 256:p // 256 + (o + q) // 256]))
    return out


def same(a, b):
    return np.array_equal(a, b, equal_nan=a.dtype.kind == "f")


LENS = {
    "one": [1], "one block": [256], "ragged": [1, 255, 256, 257, 3, 2047, 2048, 2049, 10, 4097], "zeros between": [0, 5, 0, 0, 300, 0],
    "classifier": [401408, 512, 131072, 256, 2560, 10], "thirty-three": [100 + 7 * k for k in range(33)],
    "nine hundred": [1 + (37 * k) % 700 for k in range(900)],
}


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("name", list(LENS))
@pytest.mark.parametrize("wd,decoupled", [(0.1, True), (0.01, False), (0.0, False)])
def test_steps_bit_for_bit(gpu, name, bits, wd, decoupled):
    lens = LENS[name]
    rng = np.random.default_rng(len(lens))
    exempt = [k % 3 == 1 for k in range(len(lens))]
    thetas = [rng.standard_normal(n).astype(F) for n in lens]
    stores = [gpu.from_host(t) for t in thetas]
    opt = optim.AdamMulti(gpu, stores, bits, exempt, lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=wd, decoupled=decoupled)
    plain = [Plain(n, bits) for n in lens]
    for t, scale in ((1, None), (2, 0.37), (3, None), (4, 2.0)):
        gs = grads_for(rng, lens)
        opt.set_grads([gpu.from_host(g) for g in gs])
        opt.step(t, scale)
        thetas = [p.step(th, g, t, 3e-3, 0.9, 0.99, 1e-8, wd, decoupled, e, scale) for p, th, g, e in zip(plain, thetas, gs, exempt)]
        for k, n in enumerate(lens):
            assert same(down(gpu, stores[k], n), thetas[k]), (t, k)
        for k, (p, got) in enumerate(zip(plain, state_of(gpu, opt, lens, bits))):
            want = (p.m[:p.n], p.v[:p.n]) if bits == 32 else (p.mc, p.vc, p.ms, p.vs)
            assert all(same(a, b) for a, b in zip(got, want)), (t, k)
    m, v = (down(gpu, s, opt.state_len) for s in opt.read_state())
    for k, p in enumerate(plain):
        o = opt.offset(k)
        want = p.read()
        assert same(m[o:o + p.n], want[0][:p.n]) and same(v[o:o + p.n], want[1][:p.n])


@pytest.mark.parametrize("count", [32, 33, 128, 129, 320, 321, 768, 769])
@pytest.mark.parametrize("bits", [32, 8])
def test_numbers_of_tensors_at_which_the_table_changes(gpu, count, bits):
    lens = [(97 * k) % 301 for k in range(count)]
    rng = np.random.default_rng(count)
    thetas, gs = [rng.standard_normal(n).astype(F) for n in lens], grads_for(rng, lens)
    stores = [gpu.from_host(t) if t.size else gpu.wrap_pointer(gpu.zeros(1, DType.F32).ptr, 0, DType.F32) for t in thetas]
    opt = optim.AdamMulti(gpu, stores, bits, lr=3e-3, betas=(0.9, 0.99), eps=1e-8)
    opt.set_grads([gpu.from_host(g) if g.size else None for g in gs])
    plain = [Plain(n, bits) for n in lens]
    for t in (1, 2):
        opt.step(t)
        thetas = [p.step(th, g, t, 3e-3, 0.9, 0.99, 1e-8, 0.0, False, False, None) for p, th, g in zip(plain, thetas, gs)]
    assert all(same(down(gpu, s, n), th) for s, th, n in zip(stores, thetas, lens) if n)
    want = math.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in gs))
    assert abs(float(down(gpu, opt.grad_norm(1.0)[0], 1)[0]) - want) <= 1.001 * U * want


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_32_bits_are_those_of_the_single_tensor_step(gpu, shift):
    """Tensors packed without padding, from an offset of `shift` elements, gradients at another alignment."""
    _declare(gpu.lib)
    lens = [5000, 1, 77, 4096, 12345]
    rng = np.random.default_rng(shift)
    n = sum(lens)
    th, g = rng.standard_normal(n + 8).astype(F), grads_for(rng, [n + 8])[0]
    one, many, gs = gpu.from_host(th), gpu.from_host(th), gpu.from_host(g)
    ends = np.cumsum([0] + lens)
    opt = optim.AdamMulti(gpu, [gpu.wrap_pointer(many.ptr + 4 * (int(a) + shift), k, DType.F32) for a, k in zip(ends, lens)], 32, lr=1e-2,
                          weight_decay=0.05, decoupled=True)
    opt.set_grads([gpu.wrap_pointer(gs.ptr + 4 * (int(a) + 3), k, DType.F32) for a, k in zip(ends, lens)])
    m, v = gpu.zeros(n, DType.F32), gpu.zeros(n, DType.F32)
    for t in (1, 2, 3):
        opt.step(t, 0.5)
        gpu.check(gpu.lib.wb_adam_step(gpu.handle, one.ptr + 4 * shift, gs.ptr + 12, m.ptr, v.ptr, n, t, 1e-2, 0.9, 0.999, 1e-8, 0.05, 1, 0.5))
    assert np.array_equal(down(gpu, one, n + 8), down(gpu, many, n + 8))
    mm, vv = (down(gpu, s, opt.state_len) for s in opt.read_state())
    for a, k, i in zip(ends, lens, range(len(lens))):
        o = opt.offset(i)
        assert np.array_equal(mm[o:o + k], down(gpu, m, n)[a:a + k]) and np.array_equal(vv[o:o + k], down(gpu, v, n)[a:a + k])


def test_first_step_does_not_read_the_state(gpu):
    for bits in (32, 8):
        g = gpu.from_host(np.linspace(-1, 1, 700, dtype=F))
        th = [gpu.from_host(np.ones(700, F)) for _ in range(2)]
        junk = gpu.from_host(np.full(8 * pad(700) // 4, np.nan, F))
        a = optim.AdamMulti(gpu, th[:1], bits)
        b = optim.AdamMulti(gpu, th[1:], bits, state=junk, keep_state=True)
        for o in (a, b):
            o.set_grads([g])
            o.step(1)
            o.step(2)
        assert np.array_equal(down(gpu, th[0], 700), down(gpu, th[1], 700))


@pytest.mark.parametrize("bits", [32, 8])
def test_resuming_from_the_state_bytes(gpu, bits):
    lens = [300, 4097, 12]
    rng = np.random.default_rng(bits)
    stores = [gpu.from_host(rng.standard_normal(n).astype(F)) for n in lens]
    opt = optim.AdamMulti(gpu, stores, bits, lr=1e-2)
    grads = [[gpu.from_host(g) for g in grads_for(rng, lens)] for _ in range(6)]
    for t in (1, 2, 3):
        opt.set_grads(grads[t - 1])
        opt.step(t)
    saved = [down(gpu, s, n) for s, n in zip(stores, lens)], down(gpu, opt.state, opt.state_bytes // 4)
    other = [gpu.from_host(a) for a in saved[0]]
    again = optim.AdamMulti(gpu, other, bits, lr=1e-2, state=gpu.from_host(saved[1]), keep_state=True)
    for t in (4, 5, 6):
        for o in (opt, again):
            o.set_grads(grads[t - 1])
            o.step(t)
    for a, b, n in zip(stores, other, lens):
        assert np.array_equal(down(gpu, a, n), down(gpu, b, n))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_without_gradient_is_left_alone(gpu, bits):
    lens = [600, 5, 2500]
    rng = np.random.default_rng(4)
    stores = [gpu.from_host(rng.standard_normal(n).astype(F)) for n in lens]
    opt = optim.AdamMulti(gpu, stores, bits, lr=1e-2, weight_decay=0.1, decoupled=True)
    gs = [gpu.from_host(g) for g in grads_for(rng, lens)]
    opt.set_grads(gs)
    opt.step(1)
    before = [down(gpu, s, n) for s, n in zip(stores, lens)], state_of(gpu, opt, lens, bits)
    opt.set_grads([gs[0], None, None])
    norm, _ = opt.grad_norm(1.0)
    opt.step(2)
    after = [down(gpu, s, n) for s, n in zip(stores, lens)], state_of(gpu, opt, lens, bits)
    assert not np.array_equal(before[0][0], after[0][0])
    for k in (1, 2):
        assert np.array_equal(before[0][k], after[0][k])
        assert all(np.array_equal(a, b) for a, b in zip(before[1][k], after[1][k]))
    want = math.sqrt((down(gpu, gs[0], 600).astype(np.float64) ** 2).sum())
    assert abs(down(gpu, norm, 1)[0] - want) <= 2 * U * want


def test_8_bits_stay_near_the_moments(gpu):
    """One step from zero: what is read back differs from the f32 moments by at most half the distance of two codes.  On the
    square root's scale codes are 1 / top apart, so |sqrt(x) - sqrt(x')| <= sqrt(s) (0.5 + 2 u top) / top; a root that is
    not zero may be rounded up to code 1, one whole code."""
    rng = np.random.default_rng(8)
    n = 256 * 40
    g = (rng.standard_normal(n) * np.exp(3 * rng.standard_normal(n))).astype(F)
    g[::7] = 0
    opts = [optim.AdamMulti(gpu, [gpu.zeros(n, DType.F32)], bits) for bits in (32, 8)]
    read = []
    for o in opts:
        o.set_grads([gpu.from_host(g)])
        o.step(1)
        read.append([down(gpu, s, n).astype(np.float64).reshape(-1, 256) for s in o.read_state()])
    (m, v), (m8, v8) = read
    for a, b, top, room in ((np.abs(m), np.abs(m8), 127, 0.5), (np.sqrt(v), np.sqrt(v8), 255, 1.0)):
        limit = np.sqrt(a.max(1, keepdims=True)) * (room + 4 * top * U) / top
        assert (np.abs(np.sqrt(a) - np.sqrt(b)) <= limit).all()
        big = a > a.max(1, keepdims=True) * (2 / top) ** 2
        assert (np.abs(np.sqrt(a) - np.sqrt(b)) <= limit * 0.5 / room * (1 + 1e-5))[big].all()
    assert ((v8 > 0) == (v > 0)).all() and (np.sign(m8) * np.sign(m) >= 0).all()


def test_8_bits_at_the_edges(gpu):
    """Blocks of zeros, of one value, of values near the type's ends, and blocks that are not finite, bit for bit; the last
    poison their own block alone."""
    n = 256 * 9 + 17
    g = np.zeros(n, F)
    g[256:512] = -0.5
    g[512:768] = F(1e-38)
    g[768:1024] = F(1e18)
    g[1024:1280:9] = F(1e-42)
    g[1280:1536] = np.linspace(-1e-20, 1e3, 256)
    g[1536 + 5] = np.nan
    g[1792 + 9] = np.inf
    g[2048:2304] = np.linspace(-1, 1, 256)
    g[2304:] = 3.0
    th = np.linspace(-2, 2, n, dtype=F)
    store = gpu.from_host(th)
    opt = optim.AdamMulti(gpu, [store], 8, lr=1e-2)
    opt.set_grads([gpu.from_host(g)])
    p = Plain(n, 8)
    with np.errstate(all="ignore"):
        for t in (1, 2, 3):
            opt.step(t)
            th = p.step(th, g, t, 1e-2, 0.9, 0.999, 1e-8, 0.0, False, False, None)
            assert same(down(gpu, store, n), th)
            (mc, vc, ms, vs), = state_of(gpu, opt, [n], 8)
            ok = np.isfinite(p.ms) & np.isfinite(p.vs)
            assert same(ms, p.ms) and same(vs, p.vs) and list(np.flatnonzero(~ok)) == [6, 7]
            keep = np.repeat(ok, 256)
            assert np.array_equal(mc[keep], p.mc[keep]) and np.array_equal(vc[keep], p.vc[keep])
    m, v = (down(gpu, s, pad(n)) for s in opt.read_state())
    assert np.isnan(m[1536:2048]).all() and np.isnan(v[1536:2048]).all()
    assert np.isfinite(np.delete(m, np.s_[1536:2048])).all() and np.isfinite(np.delete(v, np.s_[1536:2048])).all()


@pytest.mark.parametrize("eps", [1e-8, 0.0, 1e-30])
@pytest.mark.parametrize("scale", [1.0, 1e-12, 1e-17, 1e-20, 1e15, 1e18])
def test_8_bits_across_the_exponent_range(gpu, eps, scale):
    """Gradients from tiny to huge, eps down to 0: where the step leaves the range of its fast root and quotient it takes
    sqrt and division themselves, with the same bits."""
    rng = np.random.default_rng(3)
    n = 256 * 30 + 9
    g = (rng.standard_normal(n) * np.exp(2 * rng.standard_normal(n)) * scale).astype(F)
    th = rng.standard_normal(n).astype(F)
    store = gpu.from_host(th)
    opt = optim.AdamMulti(gpu, [store], 8, lr=1e-2, eps=eps)
    opt.set_grads([gpu.from_host(g)])
    p = Plain(n, 8)
    with np.errstate(all="ignore"):
        for t in (1, 2, 3):
            opt.step(t)
            th = p.step(th, g, t, 1e-2, 0.9, 0.999, eps, 0.0, False, False, None)
            assert same(down(gpu, store, n), th), t
            (mc, vc, ms, vs), = state_of(gpu, opt, [n], 8)
            assert same(ms, p.ms) and same(vs, p.vs), t
            # at 1e18 squares overflow: such a block's scale is NaN, it reads as NaN whatever its codes, which are not defined
            keep_m, keep_v = (np.repeat(np.isfinite(a), 256) for a in (p.ms, p.vs))
            assert same(mc[keep_m], p.mc[keep_m]) and same(vc[keep_v], p.vc[keep_v]), t


@pytest.mark.parametrize("bits", [32, 8])
def test_nothing_is_written_between_the_tensors(gpu, bits):
    """Tensors inside one guarded buffer, in another order than in memory."""
    lens, gaps = [257, 64, 3000, 1, 511], [3, 1, 70, 5, 2]
    total = sum(lens) + sum(gaps) + 9
    buf = np.full(total, -7.0, F)
    at, starts = 0, []
    for n, gap in zip(lens, gaps):
        at += gap
        starts.append(at)
        buf[at:at + n] = 0.5
        at += n
    order = [3, 0, 4, 2, 1]
    store = gpu.from_host(buf)
    size = gpu.lib
    optim._declare(size)
    need = gpu.lib.wb_adam_multi_state_bytes((ctypes.c_int64 * 5)(*[lens[k] for k in order]), 5, bits)
    room = gpu.from_host(np.full(need // 4 + 128, -7.0, F))
    opt = optim.AdamMulti(gpu, [gpu.wrap_pointer(store.ptr + 4 * starts[k], lens[k], DType.F32) for k in order], bits,
                          state=gpu.wrap_pointer(room.ptr + 256, need // 4, DType.F32))
    opt.set_grads([gpu.from_host(np.full(lens[k], 0.1, F)) for k in order])
    opt.step(1)
    opt.step(2)
    opt.grad_norm(1.0)
    opt.read_state()
    after, mask = down(gpu, store, total), np.ones(total, bool)
    for s, n in zip(starts, lens):
        mask[s:s + n] = False
        assert (after[s:s + n] < 0.5).all() and (after[s:s + n] > 0.49).all()
    assert (after[mask] == -7.0).all()
    around = down(gpu, room, need // 4 + 128)
    assert (around[:64] == -7.0).all() and (around[64 + need // 4:] == -7.0).all()


@pytest.mark.parametrize("name", list(LENS) + ["nothing"])
@pytest.mark.parametrize("scale", [1.0, 1e25, 1e-30])
def test_norm(gpu, name, scale):
    """Squares in f64 neither overflow nor vanish; the sum in f64 errs by far less than the one rounding to f32."""
    lens = [0, 0] if name == "nothing" else LENS[name]
    rng = np.random.default_rng(7)
    gs = [(g * scale).astype(F) for g in grads_for(rng, lens)]
    opt = optim.AdamMulti(gpu, [gpu.zeros(n, DType.F32) if n else gpu.wrap_pointer(gpu.zeros(1, DType.F32).ptr, 0, DType.F32) for n in lens])
    opt.set_grads([gpu.from_host(g) if g.size else None for g in gs])
    want = math.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in gs))
    for limit in (0.5, 1e30):
        got = [down(gpu, s, 1)[0] for s in opt.grad_norm(limit)]
        assert abs(float(got[0]) - want) <= 1.001 * U * want
        clip = min(1.0, limit / (want + 1e-6))
        assert abs(float(got[1]) - clip) <= 1.001 * U * clip
    first = down(gpu, opt.grad_norm(1.0)[0], 1)
    assert all(np.array_equal(first, down(gpu, opt.grad_norm(1.0)[0], 1)) for _ in range(3))


def test_norm_of_values_that_are_not_finite(gpu):
    opt = optim.AdamMulti(gpu, [gpu.zeros(1000, DType.F32)])
    for bad, norm, clip in ((np.inf, np.inf, 0.0), (np.nan, np.nan, np.nan)):
        g = np.ones(1000, F)
        g[777] = bad
        opt.set_grads([gpu.from_host(g)])
        got = [down(gpu, s, 1)[0] for s in opt.grad_norm(1.0)]
        assert np.array_equal(got, np.array([norm, clip], F), equal_nan=True)
    opt.set_grads([gpu.from_host(np.ones(1000, F))])
    assert down(gpu, opt.grad_norm(1.0)[0], 1)[0] == F(math.sqrt(1000))


@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_step(gpu, bits):
    """grad_norm's factor, read by the step on the device, is the same as that factor given by the host."""
    lens = LENS["ragged"]
    rng = np.random.default_rng(11)
    gs = [gpu.from_host(3 * g) for g in grads_for(rng, lens)]
    start = [rng.standard_normal(n).astype(F) for n in lens]
    stores = [[gpu.from_host(a) for a in start] for _ in range(2)]
    opts = [optim.AdamMulti(gpu, s, bits, lr=1e-2) for s in stores]
    for o in opts:
        o.set_grads(gs)
    for t in (1, 2):
        _, clip = opts[0].grad_norm(0.1)
        opts[0].step(t, clip)
        f = float(down(gpu, clip, 1)[0])
        assert 0 < f < 1
        opts[1].step(t, f)
    for a, b, n in zip(*stores, lens):
        assert np.array_equal(down(gpu, a, n), down(gpu, b, n))


def test_both_scales_multiply(gpu):
    g = gpu.from_host(np.linspace(-1, 1, 300, dtype=F))
    a, b = gpu.zeros(300, DType.F32), gpu.zeros(300, DType.F32)
    oa, ob = optim.AdamMulti(gpu, [a]), optim.AdamMulti(gpu, [b])
    for o in (oa, ob):
        o.set_grads([g])
    three = gpu.from_host(np.array([0.3], F))
    gpu.check(gpu.lib.wb_adam_multi_step(oa.handle, ctypes.byref(oa.config), 1, 0.7, three.ptr))
    ob.step(1, float(F(0.7) * F(0.3)))
    assert np.array_equal(down(gpu, a, 300), down(gpu, b, 300))


def test_refusals_on_a_live_handle(gpu):
    a, g = gpu.zeros(1000, DType.F32), gpu.zeros(1000, DType.F32)
    opt = optim.AdamMulti(gpu, [a], 8)
    with pytest.raises(BackendError, match="no gradients were set"):
        opt.step(1)
    with pytest.raises(BackendError, match="no gradients were set"):
        opt.grad_norm(1.0)
    with pytest.raises(BackendError, match="2 gradients for 1 tensors"):
        opt.set_grads([g, g])
    with pytest.raises(BackendError, match="overlaps"):
        opt.set_grads([a])
    with pytest.raises(BackendError, match="overlaps"):
        opt.set_grads([gpu.wrap_pointer(opt.state.ptr, 1000, DType.F32)])
    with pytest.raises(BackendError, match="gradient 0 has 10 elements"):
        opt.set_grads([gpu.zeros(10, DType.F32)])
    with pytest.raises(BackendError, match="not aligned"):
        opt.set_grads([gpu.wrap_pointer(g.ptr + 2, 1000, DType.F32)])
    with pytest.raises(BackendError, match="no gradients were set"):
        opt.step(1)
    opt.set_grads([g])
    for t in (0, -1, 2 ** 31):
        with pytest.raises(BackendError, match="counts from 1"):
            opt.step(t)
    for limit in (0.0, -1.0, float("nan")):
        with pytest.raises(BackendError, match="above 0"):
            opt.grad_norm(limit)
    one = gpu.zeros(2, DType.F32)
    with pytest.raises(BackendError, match="the two outputs are one"):
        opt.grad_norm(1.0, out=(one, one))
    with pytest.raises(BackendError, match="the two outputs are one, or not aligned"):
        opt.grad_norm(1.0, out=(gpu.wrap_pointer(one.ptr + 2, 1, DType.F32), gpu.zeros(1, DType.F32)))
    with pytest.raises(BackendError, match="scale is not aligned"):
        opt.step(1, gpu.wrap_pointer(one.ptr + 1, 1, DType.F32))
    with pytest.raises(BackendError, match="overlap"):
        opt.read_state(out=(gpu.wrap_pointer(opt.state.ptr, 1024, DType.F32), None))
    with pytest.raises(BackendError, match="two tensors"):
        optim.AdamMulti(gpu, [a, a])
    with pytest.raises(BackendError, match="no_decay"):
        optim.AdamMulti(gpu, [a], no_decay=[])
    with pytest.raises(BackendError):
        optim.AdamMulti(gpu, [])
    with pytest.raises(BackendError, match="not 16"):
        optim.AdamMulti(gpu, [a], 16)


def test_no_handle_is_made_while_the_stream_is_captured(gpu):
    import torch

    from weta_b200.backend import B200Backend

    st = torch.cuda.Stream()
    be = B200Backend(0, stream=st.cuda_stream)
    a, room = be.zeros(700, DType.F32), be.zeros(8 * pad(700) // 4, DType.F32)
    be.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        with pytest.raises(BackendError, match="being captured"):
            optim.AdamMulti(be, [a], state=room)
    del graph


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_clipped_steps(gpu, bits):
    """Norm and step captured on another stream and replayed on changing gradients equal the calls made one by one (the
    step's count is the captured one)."""
    import torch

    from weta_b200.backend import B200Backend

    lens = [4000, 33, 700]
    st = torch.cuda.Stream()
    be = B200Backend(0, stream=st.cuda_stream)
    gen = torch.Generator("cuda").manual_seed(2)
    grads = [torch.empty(n, device="cuda") for n in lens]
    arms = []
    for _ in range(2):
        th = [torch.ones(n, device="cuda") for n in lens]
        torch.cuda.synchronize()
        wrap = lambda ts: [be.wrap_pointer(t.data_ptr(), t.numel(), DType.F32) for t in ts]
        opt = optim.AdamMulti(be, wrap(th), bits, lr=1e-2)
        opt.set_grads(wrap(grads))
        arms.append((th, opt, (be.alloc(1, DType.F32), be.alloc(1, DType.F32))))

    def call(arm):
        arm[1].step(3, arm[1].grad_norm(0.5, out=arm[2])[1])

    for g in grads:
        g.normal_(generator=gen)
    torch.cuda.synchronize()
    for arm in arms:
        call(arm)
    be.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        call(arms[0])
    for _ in range(4):
        for g in grads:
            g.normal_(generator=gen)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graph.replay()
        call(arms[1])
        torch.cuda.synchronize()
        for a, b in zip(arms[0][0], arms[1][0]):
            assert torch.equal(a, b)
    del graph
    for arm in arms:
        arm[1].close()


@pytest.mark.parametrize("bits", [32, 8])
def test_scalars_may_not_lie_in_what_the_step_writes(gpu, bits):
    a, g = gpu.zeros(600, DType.F32), gpu.zeros(600, DType.F32)
    opt = optim.AdamMulti(gpu, [a], bits)
    opt.set_grads([g])
    state_end = opt.state.ptr + opt.state_bytes - 4
    for p in (a.ptr, a.ptr + 4 * 599, opt.state.ptr, state_end):
        inside, fine = gpu.wrap_pointer(p, 1, DType.F32), gpu.zeros(1, DType.F32)
        with pytest.raises(BackendError, match="lies in a parameter"):
            opt.step(1, inside)
        for out in ((inside, fine), (fine, inside)):
            with pytest.raises(BackendError, match="lies in a parameter"):
                opt.grad_norm(1.0, out=out)
    with pytest.raises(BackendError, match="bytes each"):
        opt.read_state(out=(gpu.zeros(100, DType.F32), None))
    with pytest.raises(BackendError, match="not f32"):
        optim.AdamMulti(gpu, [gpu.zeros(10, DType.F64)])
    opt.step(1, fine)
