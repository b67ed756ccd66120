"""Operators of a decoder's training step as hand-written kernels, with their gradients: norm of the query and key heads
with the position rotation in the same pass (``csrc/kernels/head_rope.cu``), causal attention over packed sequences with
grouped heads (``csrc/kernels/attention.cu``), and softmax cross entropy of a linear output layer without its logits
(``csrc/kernels/linear_ce.cu``).

They take CUDA tensors, run on the current stream of the tensors' device, and get their workspaces from torch's allocator,
so they can be captured into CUDA graphs (a backward pass, as of every torch operation, only while no eager graph of the
same leaves is alive).  Gradients are first-order and reverse-mode; other derivatives are refused.  Results and gradients do
not depend on the order in which CTAs run: repeated calls agree bit for bit.  The reference stops at the collectives
(testing/custom_implementations/work_dir/all_reduce/all_reduce_radix_batch.cpp:202); these are the operators of the
models whose gradients this package's data-parallel paths move."""
from __future__ import annotations

import ctypes as C
import struct
from functools import lru_cache

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _native as N
from ..parallel.comm import DTYPES

vp, i32, i64, f32 = C.c_void_p, C.c_int, C.c_longlong, C.c_float
N.optional("chb_matrix_status", i32, [C.POINTER(C.c_uint), vp])
N.optional("chb_matrix_status_raise", i32, [vp])
N.optional("chb_linear_ce_bytes", i32, [i64, i32, i32, C.POINTER(i64), C.POINTER(i64), C.POINTER(i64)])
N.optional("chb_linear_ce_forward", i32, [i32, vp, i64, vp, vp, i64, i32, i32, i64, i32, vp, vp, vp, vp])
N.optional("chb_linear_ce_backward", i32, [i32, vp, vp, i64, i32, i32, i32, vp, vp, vp, vp, vp])

N.optional("chb_head_rope_rows", i32, [i32, i32, C.POINTER(i32)])
N.optional("chb_head_rope", i32, [i32, vp, vp, vp, vp, i64, i32, i32, i32, vp, i32, vp, i32, f32, C.c_double, i32, vp, vp, vp])
N.optional("chb_attention_plan_bytes", i32, [i64, i32, i32, i32, C.POINTER(i64)])
N.optional("chb_attention_backward_bytes", i32, [i64, i32, i32, i32, i32, i32, C.POINTER(i64)])
N.optional("chb_attention_forward", i32, [i32, vp, vp, vp, vp, i64, i32, i32, i32, vp, i32, f32, vp, vp, vp, vp])
N.optional("chb_attention_backward", i32, [i32, vp, vp, vp, vp, vp, vp, vp, vp, i64, i32, i32, i32, i32, i32, f32, vp, vp, vp, vp, vp])

_HALF = (torch.bfloat16, torch.float16)
_ROPE_TYPES = (*_HALF, torch.float32)
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


class OperatorError(RuntimeError):
    pass


_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_functions: dict = {}
_empty_like, _contiguous = torch.empty_like, torch.contiguous_format


def _call(name: str, device: torch.device, *args) -> None:
    """One entry of the native library on the current stream of ``device``."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(N.lib(), name)
    index = device.index
    if index == _current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        raise OperatorError(f"{name} failed: {N.ERR_NAMES.get(rc, rc)}")


def _need(ok: bool, message: str):
    if not ok:
        raise ValueError(message)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, on a 16-byte boundary (copied if it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _plain(t: torch.Tensor) -> torch.Tensor:
    """The same with the strides of its shape (a dimension of one element keeps any stride otherwise)."""
    return _aligned(t).view(-1).view(t.shape)


def _new(t: torch.Tensor) -> torch.Tensor:
    """Uninitialised and contiguous, otherwise like ``t`` (half the time of torch.empty with a shape, type and device)."""
    return _empty_like(t, memory_format=_contiguous)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix whose rows are contiguous and start on 16-byte boundaries (copied if they do not)."""
    row, one = t.stride()
    if one == 1 and row % 8 == 0 and row >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return _plain(t)


def _first_order(backward):
    """A backward pass that is not differentiable itself.  Gradients are asked for without a graph nearly always, and then
    nothing of that has to be arranged."""
    slow = once_differentiable(backward)

    def run(ctx, *grads):
        if forward_ad._current_level >= 0 and any(g is not None and forward_ad.unpack_dual(g).tangent is not None for g in grads):
            raise NotImplementedError("forward-mode derivatives of a decoder operator's gradients are not implemented")
        return slow(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return staticmethod(run)


def check_operators(device=None):
    """Synchronise the current stream of ``device`` (None, or "cuda" without a number: the current device) and raise
    :class:`OperatorError` if a bounded wait inside a matrix kernel of this module ran out there since the last call (what was
    computed since then is not to be used)."""
    device = torch.device("cuda" if device is None else device)
    _need(device.type == "cuda", "check_operators: a CUDA device expected")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    word = C.c_uint(0)
    _call("chb_matrix_status", device, C.byref(word))
    if word.value:
        raise OperatorError("a wait inside a matrix kernel ran out")


def _heads(t: torch.Tensor) -> torch.Tensor:
    """[T, H, D] whose heads are contiguous and start on 16-byte boundaries (copied if they do not, and where heads or tokens
    are one in memory, as an expanded tensor's: a tensor map has no stride of zero)."""
    st, sh, one = t.stride()
    if one == 1 and st and sh and not ((st | sh) * t.element_size() | t.data_ptr()) & 15:
        return t
    return _plain(t)


_two = struct.Struct("2Q").pack        # (device pointers as a C array: packed bytes take a tenth of the time of a ctypes array)
_eight = struct.Struct("8q").pack


# ---------------------------------------------------------------------------------------- head norm and position rotation

def _head_rope(x, dy, y, heads, w, pos, eps, base, interleaved, part=None, dw=None):
    q, k = y
    a = b = c = d = e = f = g = h = 0
    if x is not None:
        (a, b, _), (c, d, _) = x[0].stride(), x[1].stride()
    if dy is not None:
        (e, f, _), (g, h, _) = dy[0].stride(), dy[1].stride()
    _call("chb_head_rope", q.device, DTYPES[q.dtype], _two(0, 0) if x is None else _two(x[0].data_ptr(), x[1].data_ptr()),
          None if dy is None else _two(dy[0].data_ptr(), dy[1].data_ptr()), _two(q.data_ptr(), k.data_ptr()), _eight(a, b, c, d, e, f, g, h),
          q.shape[0], heads[0], heads[1], q.shape[2], None if w is None else _two(w[0].data_ptr(), w[1].data_ptr()),
          0 if w is None else DTYPES[w[0].dtype], None if pos is None else pos.data_ptr(), pos is not None and pos.dtype == torch.int64,
          eps, base, interleaved, None if part is None else part.data_ptr(), None if dw is None else _two(dw[0].data_ptr(), dw[1].data_ptr()))


def _rope_forward(q, k, wq, wk, pos, eps, base, interleaved):
    y = _new(q), _new(k)
    if q.shape[0]:
        _head_rope((_heads(q), _heads(k)), None, y, (q.shape[1], k.shape[1]), None if wq is None else (_aligned(wq), _aligned(wk)), pos, eps,
                   base, interleaved)
    return y


class _HeadNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, pos, eps, base, interleaved):
        if wq is None:
            ctx.save_for_backward(pos)
        else:
            ctx.save_for_backward(pos, q, k, wq, wk)
        ctx.args = eps, base, interleaved
        return _rope_forward(q, k, wq, wk, pos, eps, base, interleaved)

    @_first_order
    def backward(ctx, gq, gk):
        saved = ctx.saved_tensors
        pos = saved[0]
        dx = _new(gq), _new(gk)
        heads = gq.shape[1], gk.shape[1]
        x = w = part = dw = None
        if len(saved) > 1:
            x, w = (_heads(saved[1]), _heads(saved[2])), (_aligned(saved[3]), _aligned(saved[4]))
            if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
                dw = torch.empty_like(w[0]), torch.empty_like(w[1])
                part = torch.empty(_rope_rows(gq.device, *heads) * gq.shape[2], dtype=torch.float32, device=gq.device)
        if gq.shape[0]:
            _head_rope(x, (_heads(gq), _heads(gk)), dx, heads, w, pos, *ctx.args, part, dw)
        elif dw:
            dw = torch.zeros_like(w[0]), torch.zeros_like(w[1])
        return (*dx, *(dw or (None, None)), None, None, None, None)


@lru_cache(maxsize=None)
def _rope_rows(device: torch.device, heads_q: int, heads_k: int) -> int:
    n = i32(0)
    with torch.cuda.device(device):
        rc = N.lib().chb_head_rope_rows(heads_q, heads_k, C.byref(n))
    if rc:
        raise OperatorError(f"chb_head_rope_rows failed: {N.ERR_NAMES.get(rc, rc)}")
    return n.value


def _wants_grad(*tensors) -> bool:
    # (inside a level of forward-mode differentiation too: torch refuses a tangent there, which a plain call would drop)
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def head_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                   positions: torch.Tensor | None = None, *, eps: float = 1e-5, base: float = 10000.0,
                   interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q`` [T, H, D] and ``k`` [T, Hk, D], then the rotation of its pairs by
    ``positions`` [T] * ``base`` ** (-2i / D), in one pass; differentiable in ``q``, ``k`` and the weights.

    bf16, fp16 or fp32; D a multiple of 8, at most 256; any strides (views of one projection's output are read in place
    where their heads start on 16-byte boundaries).  ``q_weight``, ``k_weight`` [D]: fp32 or the type of ``q``, both or
    neither (no norm then).  ``positions``: int32 or int64; None: 0, 1, 2, ...  Angles are exact to fp32's rounding within the
    turn up to positions of about 2^38 of either sign; each doubling beyond costs a bit.  ``interleaved``: pair i is elements
    2i and 2i + 1, else i and i + D / 2.  Returns contiguous tensors of the types of ``q`` and ``k``."""
    qs, ks, dtype, dev = q.shape, k.shape, q.dtype, q.device
    if len(qs) != 3 or len(ks) != 3 or qs[0] != ks[0] or qs[2] != ks[2] or qs[1] == 0 or ks[1] == 0:
        raise ValueError("head_norm_rope: q [T, H, D] and k [T, Hk, D] expected")
    if dtype not in _ROPE_TYPES or k.dtype != dtype:
        raise ValueError("head_norm_rope: q and k have to be bf16, fp16 or fp32, and alike")
    d = qs[2]
    if d % 8 or not 0 < d <= 256 or qs[0] >= 1 << 31:
        raise ValueError("head_norm_rope: D has to be a multiple of 8, at most 256")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("head_norm_rope: weights for both or for neither")
    devices = k.device == dev
    if q_weight is not None:
        if q_weight.shape != (d,) or k_weight.shape != (d,) or q_weight.dtype not in (dtype, torch.float32) or k_weight.dtype != q_weight.dtype:
            raise ValueError("head_norm_rope: weights [D] of fp32 or the type of q expected")
        devices = devices and q_weight.device == dev and k_weight.device == dev
    if positions is not None:
        if positions.shape != (qs[0],) or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("head_norm_rope: int32 or int64 positions [T] expected")
        devices = devices and positions.device == dev
        positions = positions.contiguous()
    if not (base > 0 and eps >= 0):
        raise ValueError("head_norm_rope: base has to be positive, eps not negative")
    if dev.type != "cuda" or not devices:
        raise ValueError("head_norm_rope: tensors of one CUDA device expected")
    args = q, k, q_weight, k_weight, positions, float(eps), float(base), bool(interleaved)
    return _HeadNormRope.apply(*args) if _wants_grad(q, k, q_weight, k_weight) else _rope_forward(*args)


# ------------------------------------------------------------------------------------------------------ causal attention

@lru_cache(maxsize=1024)
def _plan_bytes(T: int, group: int, seqs: int, bounds: bool) -> int:
    n = i64(0)
    rc = N.lib().chb_attention_plan_bytes(T, group, seqs, bounds, C.byref(n))
    if rc:
        raise OperatorError(f"chb_attention_plan_bytes failed: {N.ERR_NAMES.get(rc, rc)}")
    return n.value


@lru_cache(maxsize=1024)
def _backward_bytes(device: torch.device, T: int, h: int, hk: int, d: int, bounds: bool, seqs: int) -> int:
    n = i64(0)
    with torch.cuda.device(device):
        rc = N.lib().chb_attention_backward_bytes(T, h, hk, d, bounds, seqs, C.byref(n))
    if rc:
        raise OperatorError(f"chb_attention_backward_bytes failed: {N.ERR_NAMES.get(rc, rc)}")
    return n.value


def _attention_forward(q, k, v, cu, scale):
    shape, dev = q.shape, q.device
    T, h, d = shape
    hk, seqs = k.shape[1], 0 if cu is None else cu.shape[0] - 1
    o = _new(q)
    # for the backward pass: the list of work, and behind it the logarithms of the rows' sums, [h, T] fp32
    side = torch.empty(_plan_bytes(T, h // hk, seqs, cu is not None) + 4 * h * T if T else 0, dtype=torch.uint8, device=dev)
    if T:
        plan = side.data_ptr()
        q, k, v = _heads(q), _heads(k), _heads(v)
        (a, b, _), (c, e, _), (f, g, _) = q.stride(), k.stride(), v.stride()
        _call("chb_attention_forward", dev, DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), _eight(a, b, c, e, f, g, 0, 0), T, h, hk, d,
              None if cu is None else cu.data_ptr(), seqs, scale, o.data_ptr(), plan + side.shape[0] - 4 * h * T, plan)
    return o, side, -1 if cu is None else seqs


class _CausalAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, scale):
        o, side, seqs = _attention_forward(q, k, v, cu, scale)
        ctx.save_for_backward(q, k, v, o, side)      # (the bounds are in the list of work)
        ctx.args = seqs, scale
        return o

    @_first_order
    def backward(ctx, grad):
        q, k, v, o, side = ctx.saved_tensors
        seqs, scale = ctx.args
        dev = q.device
        T, h, d = q.shape
        kv = k.shape
        dq, dk, dv = _new(q), _new(k), _new(v)
        if T:
            q, k, v, grad = _heads(q), _heads(k), _heads(v), _heads(grad)
            (a, b, _), (c, e, _), (f, g, _), (m, n, _) = q.stride(), k.stride(), v.stride(), grad.stride()
            bounds, seqs = seqs >= 0, max(seqs, 0)
            work = torch.empty(_backward_bytes(dev, T, h, kv[1], d, bounds, seqs), dtype=torch.uint8, device=dev)
            _call("chb_attention_backward", dev, DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), grad.data_ptr(),
                  _eight(a, b, c, e, f, g, m, n), side.data_ptr() + side.shape[0] - 4 * h * T, side.data_ptr(), T, h, kv[1], d, bounds, seqs, scale,
                  work.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr())
        return dq, dk, dv, None, None


def causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *,
                     scale: float | None = None) -> torch.Tensor:
    """Causal softmax attention of ``q`` [T, H, D] over ``k`` and ``v`` [T, Hk, D], differentiable in all three.

    bf16 or fp16; H a multiple of Hk (head h reads key head h // (H / Hk)); D a multiple of 8, at most 128; any strides
    (views of one projection's output are read in place where their heads start on 16-byte boundaries).  ``cu_seqlens``
    [B + 1], int32 on the same device: sequence s is the rows cu_seqlens[s] to cu_seqlens[s + 1], ascending from 0 to T at
    most (not checked; bounds are clamped to 0 and T); lengths of zero are fine, rows outside all sequences get zeros and no
    gradient, and no bit of a sequence's result depends on what another holds, infinities and NaN included.  (Within a sequence
    a weight of zero times an infinity or NaN is NaN: such a value or gradient of a later token reaches the rows of its tile of
    128.)  None: one sequence.
    ``scale`` (default D ** -0.5) has to be positive.  Returns [T, H, D], contiguous."""
    qs, ks, dtype, dev = q.shape, k.shape, q.dtype, q.device
    if len(qs) != 3 or len(ks) != 3 or v.shape != ks or qs[0] != ks[0] or qs[2] != ks[2]:
        raise ValueError("causal_attention: q [T, H, D], k and v [T, Hk, D] expected")
    if dtype not in _HALF or k.dtype != dtype or v.dtype != dtype:
        raise ValueError("causal_attention: q, k and v have to be bf16 or fp16, and alike")
    h, hk, d = qs[1], ks[1], qs[2]
    if hk == 0 or h == 0 or h % hk:
        raise ValueError("causal_attention: the number of heads has to be a multiple of the key heads'")
    if d % 8 or not 0 < d <= 128:
        raise ValueError("causal_attention: D has to be a multiple of 8, at most 128")
    devices = k.device == dev and v.device == dev
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or cu_seqlens.dtype != torch.int32:
            raise ValueError("causal_attention: int32 cu_seqlens [B + 1] expected")
        devices = devices and cu_seqlens.device == dev
        cu_seqlens = cu_seqlens.contiguous()
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("causal_attention: scale has to be positive")
    if dev.type != "cuda" or not devices:
        raise ValueError("causal_attention: tensors of one CUDA device expected")
    if _wants_grad(q, k, v):
        return _CausalAttention.apply(q, k, v, cu_seqlens, scale)
    return _attention_forward(q, k, v, cu_seqlens, scale)[0]


# ---------------------------------------------------------------------------------------------- output layer and loss

@lru_cache(maxsize=256)
def _loss_bytes(device: torch.device, n: int, d: int, v: int):
    sizes = i64(0), i64(0), i64(0)
    with torch.cuda.device(device):
        rc = N.lib().chb_linear_ce_bytes(n, d, v, *(C.byref(x) for x in sizes))
    if rc:
        raise OperatorError(f"chb_linear_ce_bytes failed: {N.ERR_NAMES.get(rc, rc)}")
    return tuple(x.value for x in sizes)


def _loss_forward(x, weight, targets, ignore_index, reduction):
    (n, d), v, dev = x.shape, weight.shape[0], x.device
    kept, temporary, _ = _loss_bytes(dev, n, d, v)
    saved = torch.empty(kept, dtype=torch.uint8, device=dev)
    work = torch.empty(temporary, dtype=torch.uint8, device=dev)
    loss = torch.empty((n,) if reduction == 0 else (), dtype=torch.float32, device=dev)
    x, w, t = _rows(x), _aligned(weight), targets.contiguous()
    _call("chb_linear_ce_forward", dev, DTYPES[x.dtype], x.data_ptr(), x.stride(0), w.data_ptr(), t.data_ptr(), n, d, v, ignore_index, reduction,
          loss.data_ptr(), saved.data_ptr(), work.data_ptr())
    return loss, saved


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, ignore_index, reduction):
        loss, saved = _loss_forward(x, weight, targets, ignore_index, reduction)
        ctx.save_for_backward(weight, saved)
        ctx.args = x.shape[0], reduction
        return loss

    @_first_order
    def backward(ctx, grad):
        weight, saved = ctx.saved_tensors
        n, reduction = ctx.args
        (v, d), dev, dtype = weight.shape, weight.device, weight.dtype
        dx = torch.empty((n, d), dtype=dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty((v, d), dtype=dtype, device=dev) if ctx.needs_input_grad[1] else None
        work = torch.empty(_loss_bytes(dev, n, d, v)[2], dtype=torch.uint8, device=dev)
        w, g = _aligned(weight), grad.to(torch.float32).contiguous()
        _call("chb_linear_ce_backward", dev, DTYPES[dtype], w.data_ptr(), g.data_ptr(), n, d, v, reduction, saved.data_ptr(), work.data_ptr(),
              None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr())
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
        nothing = weight[:0].float().sum()      # (zero, and zero gradients, whatever the weight holds)
        rows = x.float().sum(-1) + nothing
        return rows if reduction == "none" else rows.sum() + nothing + (float("nan") if reduction == "mean" else 0.0)
    args = x.reshape(-1, d), weight, targets.reshape(-1), int(ignore_index), _REDUCTIONS[reduction]
    loss = _LinearCrossEntropy.apply(*args) if _wants_grad(x, weight) else _loss_forward(*args)[0]
    return loss.view(targets.shape) if reduction == "none" else loss
