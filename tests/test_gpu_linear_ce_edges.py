"""Cross entropy of a linear output layer where one row, or the size of the logits, could reach others or leave the range."""
import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb
from test_gpu_linear_ce import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_a_rows_gradient_stays_in_its_row(cuda, dtype, value):
    """dx of a row depends on that row's gradient alone."""
    x, w, t = make(150, 72, 300, dtype, 0.2)
    t[3], t[140] = 5, 6
    g = torch.Generator(device="cuda").manual_seed(9)
    grad = torch.randn(150, generator=g, device="cuda")
    grad[3], grad[140] = 0.5, -0.25                              # (neither is the largest)
    loss = chb.linear_cross_entropy(x, w, t, reduction="none")
    want, = torch.autograd.grad(loss, x, grad, retain_graph=True)
    grad[3] = value
    dx, dw = torch.autograd.grad(loss, (x, w), grad)
    keep = torch.arange(150, device="cuda") != 3
    assert torch.equal(dx[keep], want[keep])
    assert not dx[3].isfinite().any() and not dw.isfinite().any()
    grad[:] = value                                              # (all of them)
    dx, = torch.autograd.grad(chb.linear_cross_entropy(x, w, t, reduction="none"), x, grad)
    assert not dx[t != -100].isfinite().any() and not dx[t == -100].any()


def test_one_row_of_an_odd_stride(cuda):
    x, w, t = make(1, 72, 300, torch.bfloat16)
    loss = chb.linear_cross_entropy(x, w, t)
    want = loss, *torch.autograd.grad(loss, (x, w))
    wide = torch.zeros(1, 75, dtype=torch.bfloat16, device="cuda")
    wide[:, :72] = x.detach()
    wide.requires_grad_()
    loss = chb.linear_cross_entropy(wide[:, :72], w, t)
    dx, dw = torch.autograd.grad(loss, (wide, w))
    assert torch.equal(loss, want[0]) and torch.equal(dx[:, :72], want[1]) and torch.equal(dw, want[2])
