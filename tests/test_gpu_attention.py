"""Causal attention over packed sequences against the formula in 64 bits, output and gradients.

Tolerances, element by element, with u = half a step of the operands' type (eps / 2) and e = 2^-24.  A score is a sum of D
exact products in fp32; a probability is off by a factor 1 + delta, delta = 2 D e scale max sum|q||k| + 32 e (1 + max|score|)
(scores, lse, exponential).  P and dS are rounded once (u; fp16 below its normal range by 2^-25 at most, relative to a
largest probability of 1 or more), sums over n terms add (n + 16) e of the sum of sizes, results are rounded once (u).
dS = P (dP - D): dP has D e sum|dO||v|, D = sum dO O has the rounding of O, u sum|dO||O|, and D e of the same."""
import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def formula(q, k, v, do, cu, scale):
    dtype, (T, h, d), hk = q.dtype, q.shape, k.shape[1]
    u, small = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    out = [torch.zeros_like(t) for t in (q, q, k, v)]
    tol = [torch.zeros_like(t) for t in (q, q, k, v)]
    for s, e in zip(cu[:-1], cu[1:]):
        n = e - s
        if n == 0:
            continue
        sums = (n + 16) * E
        keep = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        for i in range(h):
            j = i // (h // hk)
            Q, K, V, G = q[s:e, i], k[s:e, j], v[s:e, j], do[s:e, i]
            S = (Q @ K.t() * scale).masked_fill(~keep, -float("inf"))
            P = torch.softmax(S, -1)
            delta = 2 * d * E * scale * (Q.abs() @ K.abs().t()).max() + 32 * E * (1 + S[keep].abs().max())
            O, dP = P @ V, G @ V.t()
            size = P @ V.abs()
            out[0][s:e, i], tol[0][s:e, i] = O, (u + delta + sums) * size + small * keep.double() @ V.abs() + u * O.abs()
            D = (G * O).sum(-1, keepdim=True)
            dS = P * (dP - D)
            tD = (u + d * E) * (G.abs() * O.abs()).sum(-1, keepdim=True) + (G.abs() * tol[0][s:e, i]).sum(-1, keepdim=True)
            tS = (u + sums) * dS.abs() + P * ((dP - D).abs() * delta + d * E * G.abs() @ V.abs().t() + tD) + small * keep
            out[1][s:e, i] = scale * dS @ K
            tol[1][s:e, i] = scale * tS @ K.abs() + u * out[1][s:e, i].abs()
            out[2][s:e, j] += scale * dS.t() @ Q
            tol[2][s:e, j] += scale * tS.t() @ Q.abs() + scale * (h // hk) * n * E * dS.abs().t() @ Q.abs()
            out[3][s:e, j] += P.t() @ G
            tol[3][s:e, j] += ((u + delta + (h // hk) * sums) * P + small * keep).t() @ G.abs()
    for i in (2, 3):
        tol[i] += u * out[i].abs()
    return out, [t + small for t in tol]


def make(T, h, hk, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n: torch.randn(T, n, d, generator=g, device="cuda").to(dtype)      # noqa: E731
    return r(h).requires_grad_(), r(hk).requires_grad_(), r(hk).requires_grad_(), r(h)


def bounds(lens, first=0):
    cu = [first]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def on_device(cu):
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def run(q, k, v, do, cu=None, scale=None):
    o = chb.causal_attention(q, k, v, cu, scale=scale)
    grads = torch.autograd.grad(o, (q, k, v), do)
    chb.check_operators()
    return (o.detach(), *grads)


def check(q, k, v, do, cu, scale=None):
    got = run(q, k, v, do, on_device(cu), scale)
    want, tol = formula(q, k, v, do, cu, q.shape[2] ** -0.5 if scale is None else scale)
    for name, a, b, t in zip("o dq dk dv".split(), got, want, tol):
        assert a.shape == b.shape
        assert ((a.double() - b).abs() <= t).all(), (name, ((a.double() - b).abs() - t).max())
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hk,d", [(1, 1, 8), (4, 4, 16), (2, 1, 64), (6, 2, 128), (7, 1, 40), (3, 3, 96), (5, 5, 120), (8, 1, 72)])
@pytest.mark.parametrize("lens", [[1], [127, 0, 1, 128, 129], [300, 2, 257], [640]])
def test_matches_the_formula(cuda, dtype, h, hk, d, lens):
    check(*make(sum(lens), h, hk, d, dtype, seed=sum(lens) + d), bounds(lens))


def test_many_short_sequences(cuda):
    lens = [n % 5 for n in range(150)]
    check(*make(sum(lens), 2, 2, 64, torch.bfloat16), bounds(lens))


def test_sequences_of_one_token(cuda):
    q, k, v, do = make(70, 4, 2, 64, torch.bfloat16)
    o, dq, dk, dv = check(q, k, v, do, list(range(71)))
    assert torch.equal(o, v.detach().repeat_interleave(2, 1)) and not dq.any() and not dk.any()


def test_rows_outside_all_sequences(cuda):
    q, k, v, do = make(700, 4, 2, 64, torch.bfloat16)
    cu = bounds([100, 0, 230], 133)
    want = check(q, k, v, do, cu)
    for t in want:
        assert not t[:133].any() and not t[463:].any()
    with torch.no_grad():
        for t in (q, k, v, do):
            t[:133], t[463:] = float("nan"), float("inf")
    for a, b in zip(run(q, k, v, do, on_device(cu)), want):
        assert torch.equal(a, b)


def test_no_sequence_reaches_another(cuda):
    lens = [130, 50, 200, 7]
    q, k, v, do = make(sum(lens), 6, 2, 128, torch.float16)
    cu = bounds(lens)
    want = run(q, k, v, do, on_device(cu))
    with torch.no_grad():
        for n, t in enumerate((q, k, v, do)):
            t[130:180] = float("nan") if n % 2 else float("inf")
            t[-7:] = float("inf") if n % 2 else float("nan")
    keep = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
    keep[130:180] = keep[-7:] = False
    for a, b in zip(run(q, k, v, do, on_device(cu)), want):
        assert torch.equal(a[keep], b[keep])


def test_bounds_that_lie_stay_inside(cuda):
    q, k, v, do = make(300, 2, 1, 64, torch.bfloat16)
    for cu in ([0, 5000], [-40, 300], [0, 200, 100, 300], [300, 0], [7]):
        run(q, k, v, do, on_device(cu))                       # (what is computed is not specified)
    torch.cuda.synchronize()


def test_no_bounds_is_one_sequence(cuda):
    q, k, v, do = make(333, 4, 2, 64, torch.bfloat16)
    for a, b in zip(run(q, k, v, do), run(q, k, v, do, on_device([0, 333]))):
        assert torch.equal(a, b)


def test_growing_scores_and_scale(cuda):
    """Maxima that grow by far more than 2^8 from tile to tile, and rows whose first tiles weigh nothing."""
    q, k, v, do = make(700, 2, 1, 64, torch.float16)
    with torch.no_grad():
        q.copy_(q.abs() * 0.5)
        k.copy_(k.abs() * torch.linspace(0.02, 4, 700, device="cuda")[:, None, None])
    check(q, k, v, do, [0, 700], scale=0.5)


def test_views_of_one_projection_and_odd_strides(cuda):
    T, h, hk, d = 200, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(T, (h + 2 * hk) * d, generator=g, device="cuda").bfloat16()
    parts = [t.view(T, -1, d) for t in rows.split([h * d, hk * d, hk * d], 1)]
    want = chb.causal_attention(*(t.contiguous() for t in parts))
    assert torch.equal(chb.causal_attention(*parts), want)
    odd = [torch.zeros(T, t.shape[1], d + 1, dtype=t.dtype, device="cuda") for t in parts]
    for o, t in zip(odd, parts):
        o[..., 1:] = t
    assert torch.equal(chb.causal_attention(*(t[..., 1:] for t in odd)), want)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in parts]
    assert torch.equal(chb.causal_attention(*turned), want)
    leaf = rows.clone().requires_grad_()
    o = chb.causal_attention(*(t.view(T, -1, d) for t in leaf.split([h * d, hk * d, hk * d], 1)))
    dr, = torch.autograd.grad(o.sum(), leaf)                  # (an expanded gradient)
    x = [t.contiguous().requires_grad_() for t in parts]
    dx = torch.autograd.grad(chb.causal_attention(*x), x, torch.ones(T, h, d, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(dr, torch.cat([t.reshape(T, -1) for t in dx], 1))


def test_expanded_inputs_and_gradients(cuda):
    """Heads or tokens that are one in memory (strides of zero), among queries, keys, values and gradients."""
    q, k, v, do = (t.detach() for t in make(300, 4, 4, 64, torch.bfloat16, seed=5))
    for n in range(4):
        for dim in (0, 1):
            views = [q, k, v, do]
            views[n] = views[n].narrow(dim, 0, 1).expand(300, 4, 64)
            got = [run(*(whole(t) for t in views[:3]), views[3]) for whole in (
                lambda t: t.detach().requires_grad_(), lambda t: t.contiguous().requires_grad_())]
            assert all(torch.equal(a, b) for a, b in zip(*got))
    shared = k[:, :1].clone().requires_grad_()                 # (its gradient: the sum over the heads that it was expanded to)
    dk, = torch.autograd.grad(chb.causal_attention(q, shared.expand(300, 4, 64), v), shared, do)
    whole = k[:, :1].expand(300, 4, 64).contiguous().requires_grad_()
    dw, = torch.autograd.grad(chb.causal_attention(q, whole, v), whole, do)
    assert torch.equal(dk, dw.sum(1, keepdim=True))


def test_no_tokens_and_no_sequences(cuda):
    q, k, v, do = make(0, 4, 2, 64, torch.bfloat16)
    for t in run(q, k, v, do, on_device([0])) + run(q, k, v, do):
        assert t.shape[0] == 0
    q, k, v, do = make(20, 4, 2, 64, torch.bfloat16)
    for t in run(q, k, v, do, on_device([0])):
        assert not t.any()                                    # (all rows lie outside)


def test_repeatable(cuda):
    q, k, v, do = make(1500, 8, 2, 128, torch.bfloat16)
    cu = on_device(bounds([900, 1, 599]))
    want = run(q, k, v, do, cu)
    for _ in range(5):
        for a, b in zip(run(q, k, v, do, cu), want):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits(cuda):
    T, h, d, n = (1 << 18) + 512, 64, 128, 512                # 2.15e9 elements of q
    g = torch.Generator(device="cuda").manual_seed(4)
    last = [torch.randn(n, x, d, generator=g, device="cuda").bfloat16() for x in (h, 1, 1, h)]
    big = [torch.zeros(T, x, d, dtype=torch.bfloat16, device="cuda") for x in (h, 1, 1, h)]
    for b, t in zip(big, last):
        b[-n:] = t
    for t in big[:3] + last[:3]:
        t.requires_grad_()
    cu = on_device(list(range(0, T + 1, n)))
    got = run(*big, cu)
    alone = run(*last)
    assert all(torch.equal(a[-n:], b) for a, b in zip(got[:2], alone))
    # (how many CTAs share the heads that dk and dv sum over depends on the number of tokens: another order, no other bound)
    want, tol = formula(*last, [0, n], d ** -0.5)
    for a, b, t in zip(got, want, tol):
        assert ((a[-n:].double() - b).abs() <= t).all() and not a[:-n].any()


def test_differences(cuda):
    q, k, v, do = make(150, 2, 1, 32, torch.float16)
    cu = on_device([0, 90, 150])
    o, *grads = run(q, k, v, do, cu)
    for n, leaf in enumerate((q, k, v)):
        g = torch.Generator(device="cuda").manual_seed(3 + n)
        step = torch.randint(-1, 2, leaf.shape, generator=g, device="cuda").double() * 2.0 ** -5
        f, at = [], []
        for s in (1, -1):
            args = [q.detach(), k.detach(), v.detach()]
            args[n] = (leaf.detach().double() + s * step).half()
            at.append(args[n].double())
            f.append((chb.causal_attention(*args, cu).double() * do.double()).sum())
        slope = ((at[0] - at[1]) * grads[n].double()).sum()
        # the outputs' roundings (fp16: u a value, independent) and the third order of the step
        noise = 2.0 ** -11 * (o.double() * do.double()).norm() * 12
        assert abs(f[0] - f[1] - slope) <= noise + 0.02 * abs(slope)


def test_captured_and_replayed_on_new_inputs(cuda):
    q, k, v, do = make(400, 4, 2, 64, torch.bfloat16)
    cu = on_device([0, 150, 150, 400])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = chb.causal_attention(q, k, v, cu)
        torch.autograd.grad(o, (q, k, v), do)
    torch.cuda.current_stream().wait_stream(side)
    del o
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = chb.causal_attention(q, k, v, cu)
        outs = (o.detach(), *torch.autograd.grad(o, (q, k, v), do))
    new = make(400, 4, 2, 64, torch.bfloat16, seed=8)
    with torch.no_grad():
        for a, b in zip((q, k, v, do), new):
            a.copy_(b)
    cu.copy_(on_device([0, 3, 300, 390]))                     # (the lengths are read on the device)
    graph.replay()
    for a, b in zip(outs, run(q, k, v, do, cu)):
        assert torch.equal(a, b)


def test_two_streams_at_once(cuda):
    inputs = [make(900, 4, 2, 64, torch.bfloat16, seed=i) for i in range(2)]
    cus = [on_device([0, 100, 900]), on_device([0, 33, 700, 890])]
    alone = [run(*inputs[i], cus[i]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                o = chb.causal_attention(*inputs[i][:3], cus[i])
                got[i].append((o.detach(), *torch.autograd.grad(o, inputs[i][:3], inputs[i][3])))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, alone[i]))
    chb.check_operators()


@pytest.mark.parametrize("n", [3000, 70])
def test_many_sequences_of_mixed_length(cuda, n):
    """More sequences than a warp, or a block, has threads; the first rows of a long sequence among them."""
    lens = [(i * 7919) % 11 for i in range(n)] + [777]
    q, k, v, do = make(sum(lens), 2, 1, 32, torch.float16)
    got = run(q, k, v, do, on_device(bounds(lens)))
    alone = run(*(t[-777:].detach().requires_grad_() for t in (q, k, v)), do[-777:])
    assert all(torch.equal(a[-777:], b) for a, b in zip(got[:2], alone))      # (dk and dv: summed in another order, see above)
    check(q, k, v, do, bounds(lens))


def test_gradients_of_some_inputs(cuda):
    q, k, v, do = make(200, 4, 2, 64, torch.bfloat16)
    _, dq, dk, dv = run(q, k, v, do)
    o = chb.causal_attention(q.detach(), k, v.detach())
    assert torch.equal(torch.autograd.grad(o, k, do)[0], dk)
    with pytest.raises(RuntimeError):                          # (not differentiable twice)
        g, = torch.autograd.grad(chb.causal_attention(q, k, v), q, do, create_graph=True)
        g.sum().backward()
