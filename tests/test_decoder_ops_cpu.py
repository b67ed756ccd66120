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


Q, K, W = zeros(4, 2, 16), zeros(4, 1, 16), zeros(16)


@pytest.mark.parametrize("q,k,args,kw,what", [
    (Q, K, (), {}, "CUDA device"),
    (Q, zeros(5, 1, 16), (), {}, "expected"),
    (Q, zeros(4, 0, 16), (), {}, "expected"),
    (Q, zeros(4, 1, 16, dtype=torch.float16), (), {}, "alike"),
    (Q.double(), K.double(), (), {}, "alike"),
    (zeros(4, 2, 12), zeros(4, 1, 12), (), {}, "multiple of 8"),
    (zeros(4, 2, 264), zeros(4, 1, 264), (), {}, "at most 256"),
    (Q, K, (W,), {}, "both or for neither"),
    (Q, K, (W, zeros(8)), {}, "weights"),
    (Q, K, (W, W.float()), {}, "weights"),
    (Q, K, (W.half(), W.half()), {}, "weights"),
    (Q, K, (None, None, torch.zeros(3, dtype=torch.int32)), {}, "positions"),
    (Q, K, (None, None, torch.zeros(4)), {}, "positions"),
    (Q, K, (), {"base": 0.0}, "base"),
    (Q, K, (W, W), {"eps": -1.0}, "eps"),
])
def test_head_norm_rope_refuses(q, k, args, kw, what):
    with pytest.raises(ValueError, match=what):
        chb.head_norm_rope(q, k, *args, **kw)


@pytest.mark.parametrize("q,k,v,cu,kw,what", [
    (Q, K, K, None, {}, "CUDA device"),
    (Q, K, zeros(4, 2, 16), None, {}, "expected"),
    (Q, zeros(5, 1, 16), zeros(5, 1, 16), None, {}, "expected"),
    (Q.float(), K.float(), K.float(), None, {}, "bf16 or fp16"),
    (Q, K.half(), K, None, {}, "alike"),
    (zeros(4, 3, 16), zeros(4, 2, 16), zeros(4, 2, 16), None, {}, "multiple of the key"),
    (zeros(4, 2, 12), zeros(4, 1, 12), zeros(4, 1, 12), None, {}, "multiple of 8"),
    (zeros(4, 2, 136), zeros(4, 1, 136), zeros(4, 1, 136), None, {}, "at most 128"),
    (Q, K, K, torch.zeros(2, dtype=torch.int64), {}, "cu_seqlens"),
    (Q, K, K, torch.zeros(0, dtype=torch.int32), {}, "cu_seqlens"),
    (Q, K, K, None, {"scale": 0.0}, "scale"),
    (Q, K, K, None, {"scale": float("nan")}, "scale"),
])
def test_causal_attention_refuses(q, k, v, cu, kw, what):
    with pytest.raises(ValueError, match=what):
        chb.causal_attention(q, k, v, cu, **kw)
