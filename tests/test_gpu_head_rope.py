"""Head norm and position rotation against the formula in 64 bits, outputs and gradients.

Tolerances with u = half a step of the type (eps / 2; fp32: its own 2^-24 e) and e = 2^-24: the angle is rounded to fp32
within half a turn (pi e) and its sine and cosine to fp32, so a rotated pair is off by at most 8 e of the pair's length;
a mean of D squares, its root and the products add (D + 8) e.  Together (D + 32) e |pair|, and one rounding of the result.
The sum in dx is over D terms of mixed sign: (D + 32) e of the sum of their sizes.  dw sums T * H terms in fp32, each off by
(D + 32) e, the partial sums by less than 64 additions in a row, 80 joined: (D + 256) e of the sum of the terms' sizes."""
import math

import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def formula(x, w, pos, gy, eps, base, interleaved):
    """y, dx, dw and their tolerances for one of q and k."""
    dtype, d = x.dtype, x.shape[-1]
    u, m = (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2), (d + 32) * E
    x, gy = x.detach().double(), gy.detach().double()
    i = torch.arange(d // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + d // 2)
    angle = pos.double()[:, None, None] * torch.exp(-2 * i.double() / d * math.log(base))

    def turn(z, sign):
        out, size = torch.empty_like(z), torch.empty_like(z)
        c, s = angle.cos(), sign * angle.sin()
        out[..., a], out[..., b] = z[..., a] * c - z[..., b] * s, z[..., a] * s + z[..., b] * c
        size[..., a] = size[..., b] = (z[..., a] ** 2 + z[..., b] ** 2).sqrt()
        return out, size

    r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) if w is not None else torch.ones_like(x[..., :1])
    ww = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    y, size = turn(x * r * ww, 1)
    t, tsize = turn(gy, -1)
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    ty = m * size + u * y.abs() + least
    if w is None:
        return y, t, None, ty, m * tsize + u * t.abs() + least, None
    n = x * r
    dx = r * (t * ww - n * (t * ww * n).mean(-1, keepdim=True))
    tdx = m * r * (tsize * ww.abs() + n.abs() * (tsize * ww.abs() * n.abs()).mean(-1, keepdim=True)) + u * dx.abs() + least
    dw = (t * n).sum((0, 1))
    uw = 0.0 if w.dtype == torch.float32 else torch.finfo(w.dtype).eps / 2
    tdw = (d + 256) * E * (tsize * n.abs()).sum((0, 1)) + uw * dw.abs() + least
    return y, dx, dw, ty, tdx, tdw


def make(T, h, hk, d, dtype, norm, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")      # noqa: E731
    q, k = (3 * r(T, h, d)).to(dtype).requires_grad_(), r(T, hk, d).to(dtype).requires_grad_()
    w = ((1 + 0.2 * r(d)).to(norm).requires_grad_(), (1 + 0.2 * r(d)).to(norm).requires_grad_()) if norm else (None, None)
    return q, k, *w, r(T, h, d).to(dtype), r(T, hk, d).to(dtype)


def check(q, k, wq, wk, gq, gk, pos, eps=1e-5, base=10000.0, interleaved=True):
    out = chb.head_norm_rope(q, k, wq, wk, pos, eps=eps, base=base, interleaved=interleaved)
    leaves = [t for t in (q, k, wq, wk) if t is not None]
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    p = torch.arange(len(q), device="cuda") if pos is None else pos
    for n, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        y, dx, dw, ty, tdx, tdw = formula(x, w, p, g, eps, base, interleaved)
        for got, want, tol in ((out[n], y, ty), (grads[n], dx, tdx), *(((grads[2 + n], dw, tdw),) if w is not None else ())):
            assert got.shape == want.shape
            assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() - tol).max()
    return (*out, *grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,h,hk,d,norm", [(1, 1, 1, 8, True), (1, 32, 8, 128, True), (5, 3, 1, 16, False), (33, 12, 4, 96, True),
                                           (7, 2, 2, 40, True), (19, 5, 5, 72, False), (64, 7, 1, 256, True), (300, 16, 16, 64, True),
                                           (3, 9, 3, 192, False), (2500, 6, 2, 128, True)])
def test_matches_the_formula(cuda, dtype, interleaved, T, h, hk, d, norm):
    check(*make(T, h, hk, d, dtype, dtype if norm else None, seed=T + d), None, interleaved=interleaved)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_far_negative_and_repeated_positions(cuda, kind):
    q, k, wq, wk, gq, gk = make(6, 4, 2, 64, torch.float32, torch.float32)
    pos = torch.tensor([0, -3, 1 << 20, 1 << 20, 2 ** 31 - 1, -2 ** 31], dtype=kind, device="cuda")
    if kind == torch.int64:
        pos[4] = 1 << 33
    # 64-bit angles of the formula are off by position * 2^-52 themselves: 2^-19 of a radian at 2^33, below 32 e = 2^-19
    check(q, k, wq, wk, gq, gk, pos, base=500000.0)


def test_fp32_weights_of_16_bit_heads(cuda):
    check(*make(100, 4, 2, 128, torch.bfloat16, torch.float32), None)


def test_views_of_one_projection_and_odd_strides(cuda):
    T, h, hk, d = 50, 6, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(T, (h + 2 * hk) * d, generator=g, device="cuda").bfloat16()
    q, k = rows[:, :h * d].view(T, h, d), rows[:, h * d:(h + hk) * d].view(T, hk, d)
    want = chb.head_norm_rope(q.contiguous(), k.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(chb.head_norm_rope(q, k), want))
    odd = torch.zeros(T, h, d + 3, dtype=torch.bfloat16, device="cuda")
    odd[..., 3:] = q
    turned = k.transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(a, b) for a, b in zip(chb.head_norm_rope(odd[..., 3:], turned), want))
    leaf = rows.clone().requires_grad_()
    a, b = chb.head_norm_rope(leaf[:, :h * d].view(T, h, d), leaf[:, h * d:(h + hk) * d].view(T, hk, d))
    dr, = torch.autograd.grad(a.sum() + b.sum(), leaf)            # (expanded gradients)
    x = q.clone().requires_grad_(), k.clone().requires_grad_()
    dq, dk = torch.autograd.grad(sum(t.sum() for t in chb.head_norm_rope(*x)), x)
    assert torch.equal(dr[:, :h * d].view(T, h, d), dq) and torch.equal(dr[:, h * d:(h + hk) * d].view(T, hk, d), dk)
    assert not dr[:, (h + hk) * d:].any()


def test_one_output_used_and_no_tokens(cuda):
    q, k, wq, wk, gq, gk = make(20, 4, 2, 64, torch.float32, torch.float32)
    a, _ = chb.head_norm_rope(q, k, wq, wk)
    dq, dk, dwq, dwk = torch.autograd.grad(a, (q, k, wq, wk), gq)
    full = check(q, k, wq, wk, gq, gk, None)
    assert torch.equal(dq, full[2]) and torch.equal(dwq, full[4]) and not dk.any() and not dwk.any()
    e = [t[:0].detach().requires_grad_() for t in (q, k)]
    out = chb.head_norm_rope(*e, wq, wk)
    grads = torch.autograd.grad(out, (*e, wq, wk), (gq[:0], gk[:0]))
    assert out[0].shape == (0, 4, 64) and not grads[2].any() and not grads[3].any()


def test_what_a_head_holds_stays_in_its_head(cuda):
    q, k, wq, wk, gq, gk = make(40, 4, 2, 64, torch.bfloat16, torch.float32)
    want = check(q, k, wq, wk, gq, gk, None)
    with torch.no_grad():
        k[7, 1, 3], k[9, 0, 0] = float("nan"), float("inf")
    out = chb.head_norm_rope(q, k, wq, wk)
    grads = torch.autograd.grad(out, (q, k, wq, wk), (gq, gk))
    assert torch.equal(out[0], want[0]) and torch.equal(grads[0], want[2]) and torch.equal(grads[2], want[4])
    keep = torch.ones(40, 2, dtype=torch.bool, device="cuda")
    keep[7, 1] = keep[9, 0] = False
    assert torch.equal(out[1][keep], want[1][keep]) and torch.equal(grads[1][keep], want[3][keep])
    assert grads[3].isnan().all()


def test_differences(cuda):
    q, k, wq, wk, gq, gk = make(9, 2, 1, 32, torch.float32, torch.float32)
    out = chb.head_norm_rope(q, k, wq, wk)
    grads = torch.autograd.grad(out, (q, k, wq, wk), (gq, gk))
    g = torch.Generator(device="cuda").manual_seed(2)
    for n, leaf in enumerate((q, k, wq, wk)):
        step = torch.randn(leaf.shape, generator=g, device="cuda")
        step *= 2.0 ** -8 * leaf.abs().mean() / step.abs().mean()
        f = []
        for s in (1, -1):
            args = [q, k, wq, wk]
            args[n] = (leaf + s * step).detach()
            y = chb.head_norm_rope(*args)
            f.append(sum((a.double() * b.double()).sum() for a, b in zip(y, (gq, gk))))
        slope = 2 * (step.double() * grads[n].double()).sum()
        # third order: 2^-24 of the sum of sizes, and the outputs' own error of (D + 32) e twice
        size = sum((a.double() * b.double()).abs().sum() for a, b in zip(out, (gq, gk)))
        assert abs(f[0] - f[1] - slope) <= 160 * E * size


def test_offsets_beyond_32_bits(cuda):
    T, h, d, last = 66000, 128, 256, 9                         # 2.16e9 elements of q
    g = torch.Generator(device="cuda").manual_seed(3)
    small = [torch.randn(last, n, d, generator=g, device="cuda").bfloat16() for n in (h, 1, h, 1)]
    big = [torch.zeros(T, t.shape[1], d, dtype=t.dtype, device="cuda") for t in small]
    for b, t in zip(big, small):
        b[-last:] = t
    w = torch.ones(d, device="cuda")
    pos = torch.arange(T, device="cuda", dtype=torch.int32)

    def run(q, k, gq, gk, pos):
        q.requires_grad_(), k.requires_grad_()
        out = chb.head_norm_rope(q, k, w, w, pos)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), (gq, gk)))

    for a, b in zip(run(*big, pos), run(*small, pos[-last:])):
        assert torch.equal(a[-last:], b)


def test_captured_and_replayed_on_new_inputs(cuda):
    q, k, wq, wk, gq, gk = make(300, 4, 2, 64, torch.bfloat16, torch.float32)
    pos = torch.arange(300, device="cuda")

    def step():
        out = chb.head_norm_rope(q, k, wq, wk, pos)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, (q, k, wq, wk), (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]        # (two graphs of the same call share no workspace)
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    with torch.no_grad():
        for a, b in zip((q, k, wq, wk, gq, gk), make(300, 4, 2, 64, torch.bfloat16, torch.float32, seed=4)):
            a.copy_(b)
        pos.add_(1000)
    for graph in graphs:
        graph.replay()
    want = step()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
