"""Layer norm, gradient norm and the many-tensor Adam at the edges of what their documentation allows, on the GPU."""
import numpy as np
import pytest

from weta_b200 import optim
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
