"""Head norm and rotation: strides of single tokens, and many bases in one process."""
import os

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


def resident():
    with open("/proc/self/statm") as f:
        return int(f.read().split()[1]) * os.sysconf("SC_PAGE_SIZE")


def test_bases_that_change_every_call_are_not_all_kept(cuda):
    """Rotations that are scaled with the length have a base of their own for every call."""
    q, k, *_ = make(4, 2, 1, 64, torch.bfloat16, None)
    want = chb.head_norm_rope(q.detach(), k.detach(), base=500.0)

    def calls(first, n):
        for i in range(first, first + n):
            chb.head_norm_rope(q.detach(), k.detach(), base=10000.0 + i)
        torch.cuda.synchronize()

    calls(0, 1000)
    before = resident()
    calls(1000, 15000)                                            # (16 MB of angles)
    assert resident() - before < 6 << 20
    assert all(torch.equal(a, b) for a, b in zip(chb.head_norm_rope(q.detach(), k.detach(), base=500.0), want))
