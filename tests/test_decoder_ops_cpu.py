"""What the decoder operators refuse, without a GPU."""
import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb

BF = torch.bfloat16


def zeros(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize("x,w,t,kw,what", [
    (zeros(4, 16), zeros(10, 16), zeros(4, dtype=torch.int64), {}, "CUDA device"),
    (zeros(4, 16, dtype=torch.float32), zeros(10, 16, dtype=torch.float32), zeros(4, dtype=torch.int64), {}, "bf16 or fp16"),
    (zeros(4, 16), zeros(10, 16, dtype=torch.float16), zeros(4, dtype=torch.int64), {}, "alike"),
    (zeros(4, 16), zeros(10, 16), zeros(4, dtype=torch.int32), {}, "int64"),
    (zeros(4, 16), zeros(10, 24), zeros(4, dtype=torch.int64), {}, "weight"),
    (zeros(4, 16), zeros(10, 16), zeros(5, dtype=torch.int64), {}, "target for every row"),
    (zeros(4, 12), zeros(10, 12), zeros(4, dtype=torch.int64), {}, "multiple of 8"),
    (zeros(4, 16), zeros(0, 16), zeros(4, dtype=torch.int64), {}, "out of range"),
    (zeros(4, 16), zeros(10, 16), zeros(4, dtype=torch.int64), {"reduction": "max"}, "unknown reduction"),
])
def test_linear_cross_entropy_refuses(x, w, t, kw, what):
    with pytest.raises(ValueError, match=what):
        chb.linear_cross_entropy(x, w, t, **kw)
