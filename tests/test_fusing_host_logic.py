"""CPU-only: the layer ops and the many-tensor optimizer through the fusing backend read what the plain backend would read."""
import numpy as np
import pytest

from host_backend import HostBackend
from weta_b200 import optim
from weta_b200.core import BinaryOp, DType, Layout
from weta_b200.fusion import FusingBackend

F = np.float32
N = 6
L = Layout.contiguous([N])


@pytest.fixture()
def fb():
    return FusingBackend(HostBackend())


def up(fb, a):
    return fb.inner.from_host(np.asarray(a, F))


def down(fb, s):
    return fb.to_host(s, L, DType.F32).copy()


def twice(fb, s, l=L):
    """A deferred s + s."""
    return fb.binary(BinaryOp.ADD, s, l, s, l, DType.F32)


@pytest.mark.parametrize("dropped", [False, True])
def test_a_gradient_that_shares_a_storage_keeps_its_value(fb, dropped):
    """Assigning a deferred value to a storage makes the two share it until the storage is next overwritten; an optimizer
    that was given the value still reads the value then, whether the caller kept it or not."""
    a, theta, buf = up(fb, np.arange(N)), up(fb, np.zeros(N)), up(fb, np.zeros(N))
    g = twice(fb, a)
    fb.copy_strided(g, L, DType.F32, buf, L)
    opt = optim.AdamMulti(fb, [theta])
    opt.set_grads([g])
    if dropped:
        del g
    fb.copy_strided(up(fb, np.full(N, 100)), L, DType.F32, buf, L)
    norm, _ = opt.grad_norm(1.0)
    opt.step(1)
    want = 2 * np.arange(N, dtype=F)
    assert np.array_equal(down(fb, theta), -want)
    assert fb.to_host(norm, Layout.contiguous([1]), DType.F32)[0] == F(np.sqrt((want ** 2).sum()))


def test_a_gradient_assigned_to_a_parameter_is_still_a_gradient(fb):
    """theta = g, then a step with g: the plain backend takes it, since g has a storage of its own there."""
    a, theta = up(fb, np.arange(N)), up(fb, np.zeros(N))
    opt = optim.AdamMulti(fb, [theta])
    g = twice(fb, a)
    fb.copy_strided(g, L, DType.F32, theta, L)
    opt.set_grads([g])
    opt.step(1, 0.5)
    assert np.array_equal(down(fb, theta), np.arange(N, dtype=F))
    assert np.array_equal(down(fb, g), 2 * np.arange(N, dtype=F))


def test_a_gradient_given_as_a_storage_is_read_when_the_step_runs(fb):
    theta, buf = up(fb, np.zeros(N)), up(fb, np.zeros(N))
    opt = optim.AdamMulti(fb, [theta])
    opt.set_grads([buf])
    g = twice(fb, up(fb, np.arange(N)))
    fb.copy_strided(g, L, DType.F32, buf, L)
    opt.step(1)
    assert np.array_equal(down(fb, theta), -2 * np.arange(N, dtype=F))
