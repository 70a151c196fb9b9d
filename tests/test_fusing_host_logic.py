"""CPU-only: the layer ops and the many-tensor optimizer through the fusing backend read what the plain backend would read."""
import numpy as np
import pytest

from host_backend import HostBackend
from weta_b200 import layers, optim
from weta_b200.backend import BackendError
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


def test_an_output_may_be_the_storage_that_an_operand_was_assigned_to(fb):
    """The operand's value has a storage of its own in the plain backend, so the call is no overlap and reads the old value."""
    rows = Layout.contiguous([1, N])
    a, buf = up(fb, np.arange(N)), up(fb, np.zeros(N))
    x = twice(fb, a)
    fb.copy_strided(x, L, DType.F32, buf, L)
    y, _, _ = layers.layer_norm_fwd(fb, x, rows, DType.F32, 1, out=(buf, None, None))
    assert y is buf and np.array_equal(down(fb, x), 2 * np.arange(N, dtype=F))

    dx, one = up(fb, np.zeros(N)), up(fb, np.zeros(1))
    dy = twice(fb, a)
    fb.copy_strided(dy, L, DType.F32, dx, L)
    got, _, _ = layers.layer_norm_bwd(fb, a, rows, dy, rows, DType.F32, 1, None, one, one, out=(dx, None, None))
    assert got is dx and np.array_equal(down(fb, dy), 2 * np.arange(N, dtype=F))

    work = fb.inner.alloc(16, DType.F32)
    l16 = Layout.contiguous([16])
    w = twice(fb, fb.inner.from_host(np.ones(16, F)), l16)
    fb.copy_strided(w, l16, DType.F32, work, l16)
    s, g = up(fb, np.zeros(16)), up(fb, np.zeros(16))
    layers.layer_norm_bwd(fb, s, Layout.contiguous([1, 16]), s, Layout.contiguous([1, 16]), DType.F32, 1, w, one, one, out=(None, g, None), workspace=work)
    assert np.array_equal(fb.to_host(w, l16, DType.F32), np.full(16, 2, F))


def test_nothing_of_a_closed_backend_is_used(fb):
    """Closing the wrapped backend frees what the library keeps for the optimizer's handle: it is not destroyed after that."""
    opt = optim.AdamMulti(fb, [up(fb, np.zeros(N))])
    fb.inner.close()
    assert not fb.handle
    opt.close()
    del opt
    assert "destroy" not in fb.lib.calls


@pytest.mark.parametrize("fused", [False, True])
def test_an_optimizer_of_a_closed_backend_refuses(fused):
    inner = HostBackend()
    be = FusingBackend(inner) if fused else inner
    theta, g, one, m = (inner.from_host(np.zeros(n, F)) for n in (N, N, 1, 256))
    opt = optim.AdamMulti(be, [theta])
    opt.set_grads([g])
    inner.close()
    for call in (lambda: opt.step(1), lambda: opt.step(1, one), lambda: opt.grad_norm(1.0), lambda: opt.grad_norm(1.0, out=(one, None)),
                 opt.read_state, lambda: opt.read_state(out=(m, None))):
        with pytest.raises(BackendError, match="backend is closed"):
            call()
    assert "step" not in inner.lib.calls and "read_state" not in inner.lib.calls


def test_a_deferred_operand_given_to_the_wrapped_backend(fb):
    """A deferred value has an address and a type like any storage, so the plain backend's call takes it as x and dy."""
    rows, one, y = Layout.contiguous([1, N]), up(fb, np.zeros(1)), up(fb, np.zeros(N))
    a = up(fb, np.arange(N))
    layers.layer_norm_fwd(fb.inner, twice(fb, a), rows, DType.F32, 1, out=(y, None, None))
    assert np.array_equal(down(fb, y), 2 * np.arange(N, dtype=F))
    dx = up(fb, np.zeros(N))
    layers.layer_norm_bwd(fb.inner, twice(fb, a), rows, twice(fb, y), rows, DType.F32, 1, None, one, one, out=(dx, None, None))
    assert np.array_equal(down(fb, dx), 4 * np.arange(N, dtype=F))


def test_writing_to_a_value_leaves_the_storage_it_was_assigned_to(fb):
    a, buf, nine = up(fb, np.arange(N)), up(fb, np.zeros(N)), up(fb, np.full(N, 9))
    g = twice(fb, a)
    fb.copy_strided(g, L, DType.F32, buf, L)
    fb.copy_strided(nine, L, DType.F32, g, L)
    assert np.array_equal(down(fb, g), np.full(N, 9, F)) and np.array_equal(down(fb, buf), 2 * np.arange(N, dtype=F))


@pytest.mark.parametrize("dropped", [False, True])
@pytest.mark.parametrize("how", ["copy", "layer norm", "step"])
def test_what_still_reads_a_value_is_evaluated_before_its_storage_changes(fb, how, dropped):
    """c = g + g waits while g is stored in a storage that is then written over."""
    a, buf = up(fb, np.arange(N)), up(fb, np.zeros(N))
    g = twice(fb, a)
    c = twice(fb, g)
    fb.copy_strided(g, L, DType.F32, buf, L)
    if dropped:
        del g
    if how == "copy":
        fb.copy_strided(up(fb, np.full(N, 9)), L, DType.F32, buf, L)
    elif how == "layer norm":
        layers.layer_norm_fwd(fb, up(fb, np.full(N, 9)), Layout.contiguous([1, N]), DType.F32, 1, out=(buf, None, None))
    else:
        opt = optim.AdamMulti(fb, [buf])
        opt.set_grads([up(fb, np.full(N, 9))])
        opt.step(1)
    assert np.array_equal(down(fb, c), 4 * np.arange(N, dtype=F))
    assert not np.array_equal(down(fb, buf), 2 * np.arange(N, dtype=F))


def test_what_still_reads_a_stored_value_is_evaluated_before_it_is_written_over(fb):
    g = twice(fb, up(fb, np.arange(N)))
    c = twice(fb, g)
    assert np.array_equal(down(fb, g), 2 * np.arange(N, dtype=F))
    fb.copy_strided(up(fb, np.full(N, 9)), L, DType.F32, g, L)
    assert np.array_equal(down(fb, c), 4 * np.arange(N, dtype=F)) and np.array_equal(down(fb, g), np.full(N, 9, F))


def test_nothing_is_evaluated_for_readers_that_are_gone(fb):
    a = up(fb, np.arange(N))
    g = twice(fb, a)
    c = twice(fb, twice(fb, g))  # the middle one is never stored
    down(fb, g)
    down(fb, c)
    before = fb.programs
    fb.copy_strided(a, L, DType.F32, g, L)
    assert fb.programs == before


def test_what_still_reads_a_gradient_that_got_its_own_storage(fb):
    a, theta, buf = up(fb, np.arange(N)), up(fb, np.zeros(N)), up(fb, np.zeros(N))
    g = twice(fb, a)
    c = twice(fb, g)
    fb.copy_strided(g, L, DType.F32, buf, L)
    opt = optim.AdamMulti(fb, [theta])
    opt.set_grads([g])
    fb.copy_strided(up(fb, np.full(N, 9)), L, DType.F32, g, L)
    opt.step(1)
    assert np.array_equal(down(fb, c), 4 * np.arange(N, dtype=F)) and np.array_equal(down(fb, theta), np.full(N, -9, F))
    assert np.array_equal(down(fb, buf), 2 * np.arange(N, dtype=F))
