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


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 20, 2.0 ** 34, 2.0 ** 60])
def test_logits_of_any_size(cuda, size):
    """x holds one number a row and W plain powers of two, so the logits are exact: size * (0, -1, -2, ...) / 512, or with the
    other sign.  The loss is exact but for the sum of exponentials (relative 2^-20) and one rounding."""
    v, d = 513, 8
    w = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    steps = -(torch.arange(v, device="cuda") // 64 * 64)         # (0, -64, ..., -512: eight bits are enough)
    w[:, 0] = steps / 512
    x = torch.zeros(4, d, dtype=torch.bfloat16, device="cuda")
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = size, -size, size, -size
    t = torch.tensor([0, 512, 64, 511], device="cuda")
    x, w = x.requires_grad_(), w.requires_grad_()
    loss = chb.linear_cross_entropy(x, w, t, reduction="none")
    exact = x.detach().double() @ w.detach().double().t()
    want = torch.nn.functional.cross_entropy(exact, t, reduction="none")
    assert ((loss.double() - want).abs() <= 2.0 ** -20 + 2.0 ** -24 * want.abs()).all()
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    p = torch.softmax(exact, -1)
    p[torch.arange(4, device="cuda"), t] -= 1
    # G in bf16 and results in bf16: half a step of each, and the probabilities' 2^-20; exponentials below 2^-126 are zeros, as
    # are products with them
    tiny = 2.0 ** -125
    for got, ref, scale in ((dx, p @ w.detach().double(), (p.abs() + tiny) @ w.detach().double().abs()),
                            (dw, p.t() @ x.detach().double(), (p.abs() + tiny).t() @ x.detach().double().abs())):
        assert ((got.double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -19) * (scale + ref.abs()) + 2 * tiny * (1 + size)).all()
