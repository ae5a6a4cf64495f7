"""Teachers whose logits are not all numbers."""
import pytest
import torch

import phoenix_core_b200 as pcb
from test_gpu_distill import make, reference, run

pytestmark = pytest.mark.gpu

R, Q = pcb.Algebra.REAL, pcb.Algebra.QUATERNION
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("alpha", [0.5, 1.0])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 1.7])
@pytest.mark.parametrize("algebra,dim,units", [(R, 1, 40), (Q, 4, 250), (R, 1, 40000)])
def test_nan(algebra, dim, units, temperature, alpha):
    """A NaN among a sample's entries, or in all of them, reaches its loss and the gradient of the classes that it names, and no other sample; entries of minus infinity have no
    weight, and a sample of nothing else has no second term."""
    t = torch.float32
    z, labels, teacher, index, grad = make(dim, t, 6, units, 5)
    teacher[1], teacher[2, 3], teacher[3, 0] = NAN, NAN, -INF
    teacher[4] = -INF
    teacher[5] = torch.tensor([-INF, NAN, -INF, -INF, NAN])
    want, _, size, _ = reference(z, labels, teacher, index, grad, alpha, temperature)
    loss, dz = run(dim, algebra, z, labels, teacher, index, grad, alpha, temperature)
    for row in (1, 2, 5):
        assert torch.isnan(loss[row]) and torch.isnan(dz[row, index[row]]).all(), row
        rest = torch.ones(dim * units, dtype=torch.bool)
        rest[index[row]] = False
        assert torch.isfinite(dz[row, rest]).all()
    chain = (64 + dim * units / 128) * 2.0 ** -24                    # (as in test_gpu_distill.check)
    for row in (0, 3, 4):
        assert abs(loss[row].double() - want[row]) <= chain * size[row] + 2.0 ** -24 * abs(want[row]) + 1e-37, row
        assert torch.isfinite(dz[row]).all()
