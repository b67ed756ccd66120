"""The C entries of the decoder operators refuse pointers that their kernels' words would not fit: nothing is launched, no
address is read."""
import ctypes as C
import struct

import pytest
import torch

from configurable_hierarchical_allreduce_algorithms_b200 import _native as N
from configurable_hierarchical_allreduce_algorithms_b200.ops import decoder  # noqa: F401  (declares the entries)

AT = 1 << 20                                                  # an address on every boundary that is asked for
TWO, STRIDES = struct.Struct("2Q").pack, struct.pack("8q", 64, 16, 64, 16, 64, 16, 64, 16)


def attention_forward(q=AT, k=AT, v=AT, cu=AT, o=AT, lse=AT, plan=AT):
    return N.lib().chb_attention_forward(N.BF16, q, k, v, STRIDES, 4, 4, 4, 16, cu, 1, 1.0, o, lse, plan, None)


def attention_backward(q=AT, k=AT, v=AT, o=AT, dout=AT, lse=AT, plan=AT, work=AT, dq=AT, dk=AT, dv=AT):
    return N.lib().chb_attention_backward(N.F16, q, k, v, o, dout, STRIDES, lse, plan, 4, 4, 4, 16, 1, 1, 1.0, work, dq, dk, dv, None)


def head_rope(q=AT, gq=AT, y=AT, w=AT, pos=AT, part=AT, dw=AT):
    return N.lib().chb_head_rope(N.BF16, TWO(q, AT), TWO(gq, AT), TWO(y, AT), STRIDES, 4, 4, 4, 16, TWO(w, AT), N.F32, pos, 1, 1e-5, 1e4, 1,
                                 part, TWO(dw, AT), None)


def loss_forward(x=AT, w=AT, targets=AT, loss=AT, saved=AT, work=AT):
    return N.lib().chb_linear_ce_forward(N.BF16, x, 16, w, targets, 4, 16, 10, -100, 1, loss, saved, work, None)


def loss_backward(w=AT, grad=AT, saved=AT, work=AT, dx=AT, dw=AT):
    return N.lib().chb_linear_ce_backward(N.BF16, w, grad, 4, 16, 10, 1, saved, work, dx, dw, None)


@pytest.mark.parametrize("entry,names", [
    (attention_forward, {"q": 8, "k": 8, "v": 2, "cu": 2, "o": 8, "lse": 2, "plan": 8}),
    (attention_backward, {"q": 8, "k": 8, "v": 8, "o": 8, "dout": 2, "lse": 1, "plan": 4, "work": 8, "dq": 8, "dk": 2, "dv": 8}),
    (head_rope, {"q": 8, "gq": 8, "y": 8, "w": 4, "pos": 4, "part": 2, "dw": 2}),
    (loss_forward, {"x": 8, "w": 8, "targets": 4, "loss": 2, "saved": 8, "work": 8}),
    (loss_backward, {"w": 8, "grad": 2, "saved": 8, "work": 16, "dx": 8, "dw": 8}),
])
def test_pointers_off_their_boundary_are_refused(entry, names):
    for name, off in names.items():
        assert entry(**{name: AT + off}) == N.ERR_ARG, name
    if not torch.cuda.is_available():                         # (with a device these calls would launch)
        assert entry() == N.ERR_CUDA
    assert C.sizeof(C.c_void_p) == 8
