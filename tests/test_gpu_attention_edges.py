"""Causal attention where strides, the type's range, other sequences or masked keys could reach a result: against the formula in
64 bits (tolerances: see test_gpu_attention.py) or against a call that has to agree bit for bit."""
import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb
from test_gpu_attention import bounds, formula, make, on_device, run

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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_large_neighbours_change_no_rounding(cuda, dtype, d):
    """The next sequence's queries lie in this one's last tile; what they are changes no bit of this one's results."""
    lens = [300, 200]
    q, k, v, do = make(500, 4, 2, d, dtype, seed=6)
    with torch.no_grad():
        k[:300] *= torch.linspace(0.5, 2, 300, device="cuda")[:, None, None]      # (maxima that grow by less than 2^8)
    cu = on_device(bounds(lens))
    want = run(q, k, v, do, cu)
    with torch.no_grad():
        for t in (q, k, v, do):
            t[300:] *= 100
    for a, b in zip(run(q, k, v, do, cu), want):
        assert torch.equal(a[:300], b[:300])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_keys_ruled_out_by_infinities(cuda, dtype, d):
    """A document whose first keys are padding, ruled out by minus infinity in one place: whole tiles without a weight."""
    q, k, v, _ = make(400, 2, 1, d, dtype, seed=7)
    q, k, v = q.detach(), k.detach(), v.detach()
    q[..., 0], q[..., 1] = 1, 30
    k[:150, :, 0], k[150:, :, 0], k[150:, :, 1] = -float("inf"), 0, -30
    got = chb.causal_attention(q, k, v)
    want, tol = formula(q[150:], k[150:], v[150:], torch.zeros_like(q[150:]), [0, 250], d ** -0.5)
    assert ((got[150:].double() - want[0]).abs() <= tol[0]).all()
    assert got[:150].isnan().all()                               # (no key at all)
