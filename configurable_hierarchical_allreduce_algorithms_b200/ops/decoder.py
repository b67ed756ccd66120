"""Operators of a decoder's training step as hand-written kernels, with their gradients: norm of the query and key heads
with the position rotation in the same pass (``csrc/kernels/head_rope.cu``), causal attention over packed sequences with
grouped heads (``csrc/kernels/attention.cu``), and softmax cross entropy of a linear output layer without its logits
(``csrc/kernels/linear_ce.cu``).

They take CUDA tensors, run on the current stream of the tensors' device, and get their workspaces from torch's allocator,
so they can be captured into CUDA graphs.  The reference stops at the collectives
(testing/custom_implementations/work_dir/all_reduce/all_reduce_radix_batch.cpp:202); these are the operators of the
models whose gradients this package's data-parallel paths move."""
from __future__ import annotations

import contextlib
import ctypes as C
import struct
from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N
from ..parallel.comm import DTYPES

vp, i32, i64, f32 = C.c_void_p, C.c_int, C.c_longlong, C.c_float
N.optional("chb_matrix_status", i32, [C.POINTER(C.c_uint), vp])
N.optional("chb_linear_ce_bytes", i32, [i64, i32, i32, C.POINTER(i64), C.POINTER(i64), C.POINTER(i64)])
N.optional("chb_linear_ce_forward", i32, [i32, vp, i64, vp, vp, i64, i32, i32, i64, i32, vp, vp, vp, vp])
N.optional("chb_linear_ce_backward", i32, [i32, vp, vp, i64, i32, i32, i32, vp, vp, vp, vp, vp])

N.optional("chb_head_rope_rows", i32, [i32, i32, C.POINTER(i32)])
N.optional("chb_head_rope", i32, [i32, vp, vp, vp, vp, i64, i32, i32, i32, vp, i32, vp, i32, f32, C.c_double, i32, vp, vp, vp])
N.optional("chb_attention_forward", i32, [i32, vp, vp, vp, vp, i64, i32, i32, i32, vp, i32, f32, vp, vp, vp])
N.optional("chb_attention_backward", i32, [i32, vp, vp, vp, vp, vp, vp, vp, i64, i32, i32, i32, vp, i32, f32, vp, vp, vp, vp, vp])

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


def _heads(t: torch.Tensor) -> torch.Tensor:
    """[T, H, D] whose heads are contiguous and start on 16-byte boundaries (copied if they do not)."""
    size = t.element_size()
    if t.stride(2) == 1 and all(t.stride(i) * size % 16 == 0 for i in (0, 1)) and t.data_ptr() % 16 == 0:
        return t
    return _aligned(t)


def _table(*tensors) -> bytes:
    """Device pointers as a C array (packed bytes: a tenth of the time of a ctypes array)."""
    return _pack_table[len(tensors)](*[0 if t is None else t.data_ptr() for t in tensors])


_pack_table = {k: struct.Struct(f"{k}Q").pack for k in (2,)}
_pack_strides = struct.Struct("8q").pack


# ---------------------------------------------------------------------------------------- head norm and position rotation

def _head_rope(x, dy, y, heads, w, pos, eps, base, interleaved, part=None, dw=None):
    q, k = y
    sx, sd = (((t.stride(0), t.stride(1)) if t is not None else (0, 0) for t in ts) for ts in (x, dy or (None, None)))
    (a, b), (c, d) = sx
    (e, f), (g, h) = sd
    dev = q.device
    with _on(dev):
        rc = N.lib().chb_head_rope(DTYPES[q.dtype], _table(*x), _table(*dy) if dy else None, _table(q, k), _pack_strides(a, b, c, d, e, f, g, h),
                                   q.shape[0], heads[0], heads[1], q.shape[2], _table(*w) if w else None,
                                   DTYPES[w[0].dtype] if w else 0, pos.data_ptr() if pos is not None else None,
                                   int(pos is not None and pos.dtype == torch.int64), eps, base, interleaved,
                                   part.data_ptr() if part is not None else None, _table(*dw) if dw else None, _stream(dev))
    _check(rc, "head_norm_rope")


class _HeadNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, pos, eps, base, interleaved):
        heads = q.shape[1], k.shape[1]
        x = _heads(q), _heads(k)
        y = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
        w = None if wq is None else (_aligned(wq), _aligned(wk))
        if len(q):
            _head_rope(x, None, y, heads, w, pos, eps, base, interleaved)
        ctx.normed = w is not None
        ctx.save_for_backward(*((q, k, wq, wk) if w else ()), *((pos,) if pos is not None else ()))
        ctx.args = eps, base, interleaved, pos is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        eps, base, interleaved, has_pos = ctx.args
        saved = ctx.saved_tensors
        pos = saved[-1] if has_pos else None
        dy = _heads(gq), _heads(gk)
        heads = gq.shape[1], gk.shape[1]
        dx = torch.empty(gq.shape, dtype=gq.dtype, device=gq.device), torch.empty(gk.shape, dtype=gk.dtype, device=gk.device)
        x, w, part, dw = (None, None), None, None, None
        if ctx.normed:
            x, w = (_heads(saved[0]), _heads(saved[1])), (_aligned(saved[2]), _aligned(saved[3]))
            if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
                dw = torch.empty_like(w[0]), torch.empty_like(w[1])
                part = torch.empty(_rope_rows(gq.device, *heads) * gq.shape[2], dtype=torch.float32, device=gq.device)
        if len(gq):
            _head_rope(x, dy, dx, heads, w, pos, eps, base, interleaved, part, dw)
        elif dw:
            dw = torch.zeros_like(w[0]), torch.zeros_like(w[1])
        return (*dx, *(dw or (None, None)), None, None, None, None)


@lru_cache(maxsize=None)
def _rope_rows(device: torch.device, heads_q: int, heads_k: int) -> int:
    n = i32(0)
    with _on(device):
        _check(N.lib().chb_head_rope_rows(heads_q, heads_k, C.byref(n)), "chb_head_rope_rows")
    return n.value


def head_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                   positions: torch.Tensor | None = None, *, eps: float = 1e-5, base: float = 10000.0,
                   interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q`` [T, H, D] and ``k`` [T, Hk, D], then the rotation of its pairs by
    ``positions`` [T] * ``base`` ** (-2i / D), in one pass; differentiable in ``q``, ``k`` and the weights.

    bf16, fp16 or fp32; D a multiple of 8, at most 256; any strides (views of one projection's output are read in place
    where their heads start on 16-byte boundaries).  ``q_weight``, ``k_weight`` [D]: fp32 or the type of ``q``, both or
    neither (no norm then).  ``positions``: int32 or int64, any value; None: 0, 1, 2, ...  ``interleaved``: pair i is
    elements 2i and 2i + 1, else i and i + D / 2.  Returns contiguous tensors of the types of ``q`` and ``k``."""
    _need(q.dim() == 3 and k.dim() == 3 and q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2] and q.shape[1] > 0 and k.shape[1] > 0,
          "head_norm_rope: q [T, H, D] and k [T, Hk, D] expected")
    _need(q.dtype in (*_HALF, torch.float32) and k.dtype == q.dtype, "head_norm_rope: q and k have to be bf16, fp16 or fp32, and alike")
    d = q.shape[2]
    _need(d % 8 == 0 and 0 < d <= 256 and q.shape[0] < 1 << 31, "head_norm_rope: D has to be a multiple of 8, at most 256")
    _need((q_weight is None) == (k_weight is None), "head_norm_rope: weights for both or for neither")
    tensors = [q, k]
    if q_weight is not None:
        tensors += [q_weight, k_weight]
        _need(all(w.shape == (d,) and w.dtype in (q.dtype, torch.float32) for w in tensors[2:]) and q_weight.dtype == k_weight.dtype,
              "head_norm_rope: weights [D] of fp32 or the type of q expected")
    if positions is not None:
        tensors.append(positions)
        _need(positions.shape == (q.shape[0],) and positions.dtype in (torch.int32, torch.int64),
              "head_norm_rope: int32 or int64 positions [T] expected")
    _need(base > 0 and eps >= 0, "head_norm_rope: base has to be positive, eps not negative")
    _need(q.is_cuda and all(t.device == q.device for t in tensors), "head_norm_rope: tensors of one CUDA device expected")
    return _HeadNormRope.apply(q, k, q_weight, k_weight, None if positions is None else positions.contiguous(), float(eps),
                               float(base), bool(interleaved))


# ------------------------------------------------------------------------------------------------------ causal attention

def _strides(*tensors) -> bytes:
    s = [x for t in tensors for x in (t.stride(0), t.stride(1))]
    return _pack_strides(*s, *(0,) * (8 - len(s)))


class _CausalAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, scale):
        T, h, d = q.shape
        o = torch.empty(T, h, d, dtype=q.dtype, device=q.device)
        lse = torch.empty(h, T, dtype=torch.float32, device=q.device)
        if T:
            qs, ks, vs = _heads(q), _heads(k), _heads(v)
            with _on(q.device):
                rc = N.lib().chb_attention_forward(DTYPES[q.dtype], qs.data_ptr(), ks.data_ptr(), vs.data_ptr(), _strides(qs, ks, vs), T, h,
                                                   k.shape[1], d, cu.data_ptr() if cu is not None else None,
                                                   cu.numel() - 1 if cu is not None else 0, scale, o.data_ptr(), lse.data_ptr(),
                                                   _stream(q.device))
            _check(rc, "causal_attention")
        ctx.save_for_backward(q, k, v, o, lse, *(() if cu is None else (cu,)))
        ctx.scale = scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, o, lse, *rest = ctx.saved_tensors
        cu = rest[0] if rest else None
        T, h, d = q.shape
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        if T:
            qs, ks, vs, g = _heads(q), _heads(k), _heads(v), _heads(grad)
            delta = torch.empty(h, T, dtype=torch.float32, device=q.device)
            with _on(q.device):
                rc = N.lib().chb_attention_backward(DTYPES[q.dtype], qs.data_ptr(), ks.data_ptr(), vs.data_ptr(), o.data_ptr(), g.data_ptr(),
                                                    _strides(qs, ks, vs, g), lse.data_ptr(), T, h, k.shape[1], d,
                                                    cu.data_ptr() if cu is not None else None, cu.numel() - 1 if cu is not None else 0,
                                                    ctx.scale, delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                                    _stream(q.device))
            _check(rc, "causal_attention backward")
        return dq, dk, dv, None, None


def causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *,
                     scale: float | None = None) -> torch.Tensor:
    """Causal softmax attention of ``q`` [T, H, D] over ``k`` and ``v`` [T, Hk, D], differentiable in all three.

    bf16 or fp16; H a multiple of Hk (head h reads key head h // (H / Hk)); D a multiple of 8, at most 128; any strides
    (views of one projection's output are read in place where their heads start on 16-byte boundaries).  ``cu_seqlens``
    [B + 1], int32 on the same device: sequence s is the rows cu_seqlens[s] to cu_seqlens[s + 1], ascending from 0 to T at
    most (not checked; bounds are clamped to 0 and T); lengths of zero are fine, rows outside all sequences get zeros and no
    gradient, and no sequence is reached by what another holds, infinities and NaN included.  None: one sequence.
    ``scale`` (default D ** -0.5) has to be positive.  Returns [T, H, D], contiguous."""
    _need(q.dim() == 3 and k.dim() == 3 and v.shape == k.shape and q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2],
          "causal_attention: q [T, H, D], k and v [T, Hk, D] expected")
    _need(q.dtype in _HALF and k.dtype == q.dtype and v.dtype == q.dtype, "causal_attention: q, k and v have to be bf16 or fp16, and alike")
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    _need(hk > 0 and h > 0 and h % hk == 0, "causal_attention: the number of heads has to be a multiple of the key heads'")
    _need(d % 8 == 0 and 0 < d <= 128, "causal_attention: D has to be a multiple of 8, at most 128")
    if cu_seqlens is not None:
        _need(cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 1 and cu_seqlens.dtype == torch.int32, "causal_attention: int32 cu_seqlens [B + 1] expected")
    scale = d ** -0.5 if scale is None else float(scale)
    _need(0.0 < scale < float("inf"), "causal_attention: scale has to be positive")
    _need(q.is_cuda and all(t.device == q.device for t in (k, v, cu_seqlens) if t is not None), "causal_attention: tensors of one CUDA device expected")
    return _CausalAttention.apply(q, k, v, None if cu_seqlens is None else cu_seqlens.contiguous(), scale)


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
