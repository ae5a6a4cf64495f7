"""Gradients through the residual path of a block whose norm behind it nobody used."""
import pytest
import torch

import phoenix_core_b200 as pcb
from phoenix_core_b200.autograd import QResidualNorm, ResidualNormFunction

pytestmark = pytest.mark.gpu

R = pcb.Algebra.REAL


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("f", [64, 130, 8200])
def test_values_that_are_not_finite_stay_where_they_are(dtype, f):
    """The residual's gradient is that of y, whatever y holds: an infinity or a NaN in a row is no part of it."""
    gen = torch.Generator().manual_seed(f)
    x = torch.randn((6, f), generator=gen).to(dtype).cuda()
    x[0, 3], x[2, f - 1], x[4] = float("inf"), float("nan"), float("-inf")
    branch, grad = torch.randn((6, f), generator=gen).to(dtype).cuda(), torch.randn((6, f), generator=gen).to(dtype).cuda()
    pre, post = torch.ones(f, device="cuda", requires_grad=True), (torch.rand(f, generator=gen) + 0.5).cuda().requires_grad_(True)
    x.requires_grad_(True)
    branch.requires_grad_(True)
    y, h = ResidualNormFunction.apply(x, branch, None, post, pre, R)
    del h
    y.backward(grad)
    assert torch.equal(x.grad, grad) and torch.isfinite(branch.grad).all() and torch.isfinite(post.grad).all() and (pre.grad == 0).all()
    clean = [t.detach().clone().requires_grad_(True) for t in (torch.randn_like(x), branch, post, pre)]
    y, _ = ResidualNormFunction.apply(clean[0], clean[1], None, clean[2], clean[3], R)
    y.backward(grad)
    assert torch.equal(clean[1].grad, branch.grad) and torch.equal(clean[2].grad, post.grad)       # (they do not depend on x)


def test_in_front_of_a_block():
    """Without a branch y is the residual itself."""
    layer = QResidualNorm(48, R)
    x = torch.randn((5, 48), device="cuda")
    x[1, 1] = float("inf")
    x.requires_grad_(True)
    y, h = layer(x)
    (y * 3.0).sum().backward()
    assert (x.grad == 3.0).all() and (layer.pre_weight.grad == 0).all()
