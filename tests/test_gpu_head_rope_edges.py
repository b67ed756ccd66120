"""Head norm and rotation: strides of single tokens."""
import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb
from test_gpu_head_rope import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_token_of_odd_strides(cuda, dtype):
    """A dimension of one element may have any stride: it is never taken."""
    q, k, wq, wk, gq, gk = make(1, 4, 2, 64, dtype, torch.float32)
    want = check(q, k, wq, wk, gq, gk, None)
    odd = []
    for t in (q, k, gq, gk):
        rows = torch.zeros(1, t.numel() + 3, dtype=t.dtype, device="cuda")
        rows[:, :t.numel()] = t.detach().flatten()
        odd.append(rows.as_strided(t.shape, (t.numel() + 3, 64, 1)))
    a, b = (t.detach().requires_grad_() for t in odd[:2])
    out = chb.head_norm_rope(a, b, wq, wk)
    grads = torch.autograd.grad(out, (a, b, wq, wk), odd[2:])
    assert all(torch.equal(p, r) for p, r in zip((*out, *grads), want))
    one = q.detach()[:, :1].as_strided((1, 1, 64), (64, 3, 1))
    assert torch.equal(chb.head_norm_rope(one, one)[0], chb.head_norm_rope(one.clone(), one.clone())[0])
