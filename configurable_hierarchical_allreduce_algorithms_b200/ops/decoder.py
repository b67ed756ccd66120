"""Operators of a decoder's training step as hand-written kernels, with their gradients: softmax cross entropy of a linear
output layer without its logits (``csrc/kernels/linear_ce.cu``).

They take CUDA tensors, run on the current stream of the tensors' device, and get their workspaces from torch's allocator,
so they can be captured into CUDA graphs.  The reference stops at the collectives
(testing/custom_implementations/work_dir/all_reduce/all_reduce_radix_batch.cpp:202); these are the operators of the
models whose gradients this package's data-parallel paths move."""
from __future__ import annotations

import contextlib
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N
from ..parallel.comm import DTYPES

vp, i32, i64, f32 = C.c_void_p, C.c_int, C.c_longlong, C.c_float
N.optional("chb_matrix_status", i32, [C.POINTER(C.c_uint), vp])
N.optional("chb_linear_ce_bytes", i32, [i64, i32, i32, C.POINTER(i64), C.POINTER(i64), C.POINTER(i64)])
N.optional("chb_linear_ce_forward", i32, [i32, vp, i64, vp, vp, i64, i32, i32, i64, i32, vp, vp, vp, vp])
N.optional("chb_linear_ce_backward", i32, [i32, vp, vp, i64, i32, i32, i32, vp, vp, vp, vp, vp])

_HALF = (torch.bfloat16, torch.float16)
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


class OperatorError(RuntimeError):
    pass


def _check(rc: int, what: str):
    if rc:
        raise OperatorError(f"{what} failed: {N.ERR_NAMES.get(rc, rc)}")


def _on(device: torch.device):
    """Makes ``device`` current for a launch if it is not."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _need(ok: bool, message: str):
    if not ok:
        raise ValueError(message)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, on a 16-byte boundary (copied if it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix whose rows are contiguous and start on 16-byte boundaries (copied if they do not)."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return _aligned(t)


def check_operators(device=None):
    """Synchronise the current stream and raise :class:`OperatorError` if a bounded wait inside a matrix kernel of this
    module ran out since the last call (its outputs are not to be used then)."""
    device = torch.device("cuda", torch.cuda.current_device() if device is None else torch.device(device).index or 0)
    with _on(device):
        word = C.c_uint(0)
        _check(N.lib().chb_matrix_status(C.byref(word), _stream(device)), "chb_matrix_status")
    if word.value:
        raise OperatorError("a wait inside a matrix kernel ran out")


# ---------------------------------------------------------------------------------------------- output layer and loss

class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, ignore_index, reduction):
        n, d = x.shape
        v = weight.shape[0]
        sizes = (i64 * 3)()
        at = C.addressof(sizes)
        ptr = lambda i: C.cast(at + 8 * i, C.POINTER(i64))      # noqa: E731
        lib, code = N.lib(), DTYPES[x.dtype]
        _check(lib.chb_linear_ce_bytes(n, d, v, ptr(0), ptr(1), ptr(2)), "chb_linear_ce_bytes")
        byte = lambda k: torch.empty(k, dtype=torch.uint8, device=x.device)     # noqa: E731
        saved, work = byte(sizes[0]), byte(sizes[1])
        loss = torch.empty(n if reduction == 0 else (), dtype=torch.float32, device=x.device)
        xr, w, t = _rows(x), _aligned(weight), targets.contiguous()
        with _on(x.device):
            rc = lib.chb_linear_ce_forward(code, xr.data_ptr(), xr.stride(0), w.data_ptr(), t.data_ptr(), n, d, v, ignore_index,
                                           reduction, loss.data_ptr(), saved.data_ptr(), work.data_ptr(), _stream(x.device))
        _check(rc, "linear_cross_entropy")
        ctx.save_for_backward(weight, saved)
        ctx.sizes = n, d, v, sizes[2], reduction, code
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        weight, saved = ctx.saved_tensors
        n, d, v, nbytes, reduction, code = ctx.sizes
        dev = weight.device
        dx = torch.empty(n, d, dtype=weight.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty(v, d, dtype=weight.dtype, device=dev) if ctx.needs_input_grad[1] else None
        work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        w, g = _aligned(weight), grad.to(torch.float32).contiguous()
        with _on(dev):
            rc = N.lib().chb_linear_ce_backward(code, w.data_ptr(), g.data_ptr(), n, d, v, reduction, saved.data_ptr(),
                                                work.data_ptr(), dx.data_ptr() if dx is not None else None,
                                                dw.data_ptr() if dw is not None else None, _stream(dev))
        _check(rc, "linear_cross_entropy backward")
        return dx, dw, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """``cross_entropy(x @ weight.T, targets)`` without the logits, differentiable in ``x`` and ``weight``.

    ``x`` [..., D] and ``weight`` [V, D]: bf16 or fp16, D a multiple of 8; ``targets`` [...]: int64 labels.  A row whose label
    is ``ignore_index`` has a loss of zero, is not counted by the mean and costs nothing; whatever its ``x`` holds reaches
    nothing else.  A label outside the vocabulary makes its row's loss, and the gradients that depend on it, NaN.
    Returns fp32: a scalar ("mean" over the labelled rows, NaN without any; "sum"), or [...] ("none")."""
    _need(x.dtype in _HALF and weight.dtype == x.dtype, "linear_cross_entropy: x and weight have to be bf16 or fp16, and alike")
    _need(targets.dtype == torch.int64, "linear_cross_entropy: int64 targets expected")
    _need(weight.dim() == 2 and x.dim() >= 1 and x.shape[-1] == weight.shape[1], "linear_cross_entropy: x [..., D] and weight [V, D] expected")
    _need(targets.shape == x.shape[:-1], "linear_cross_entropy: a target for every row of x expected")
    d, v = weight.shape[1], weight.shape[0]
    _need(d % 8 == 0 and d > 0, "linear_cross_entropy: D has to be a multiple of 8")
    _need(0 < v < 1 << 30 and targets.numel() < (1 << 31) - 256, "linear_cross_entropy: vocabulary or number of rows out of range")
    _need(reduction in _REDUCTIONS, f"linear_cross_entropy: unknown reduction {reduction!r}")
    _need(x.is_cuda and weight.device == x.device and targets.device == x.device, "linear_cross_entropy: tensors of one CUDA device expected")
    if targets.numel() == 0:
        zero = x.float().sum() + 0.0 * weight[:1].float().sum()
        return x.float().sum(-1) if reduction == "none" else zero / 0.0 if reduction == "mean" else zero
    loss = _LinearCrossEntropy.apply(x.reshape(-1, d), weight, targets.reshape(-1), int(ignore_index), _REDUCTIONS[reduction])
    return loss.view(targets.shape) if reduction == "none" else loss
