"""Causal attention where strides, the type's range, other sequences or masked keys could reach a result: against the formula in
64 bits (tolerances: see test_gpu_attention.py) or against a call that has to agree bit for bit."""
import pytest
import torch

from test_gpu_attention import make, run

pytestmark = pytest.mark.gpu


def test_one_token_of_odd_strides(cuda):
    """A dimension of one element may have any stride: it is never taken."""
    q, k, v, do = make(1, 4, 2, 64, torch.bfloat16, seed=8)
    want = run(q, k, v, do)
    odd = []
    for t in (q, k, v, do):
        rows = torch.zeros(1, t.numel() + 3, dtype=t.dtype, device="cuda")
        rows[:, :t.numel()] = t.detach().flatten()
        odd.append(rows.as_strided(t.shape, (t.numel() + 3, 64, 1)))
    odd[:3] = [t.detach().requires_grad_() for t in odd[:3]]
    assert all(torch.equal(a, b) for a, b in zip(run(*odd), want))
