"""Causal attention where strides, the type's range, other sequences or masked keys could reach a result: against the formula in
64 bits (tolerances: see test_gpu_attention.py) or against a call that has to agree bit for bit."""
import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb
from test_gpu_attention import bounds, check, formula, make, on_device, run

pytestmark = pytest.mark.gpu


def in_eighths(t):
    """Multiples of 1/8, at most 2: any power of two times them is exact from 2^-21 on."""
    return (t.detach().float().clamp(-2, 2) * 8).round().div(8)


def test_one_token_of_odd_strides(cuda):
    """A dimension of one element may have any stride: it is never taken."""
    q, k, v, do = make(1, 4, 2, 64, torch.bfloat16, seed=8)
    want = run(q, k, v, do)
    odd = []
    for t in (q, k, v, do):
        rows = torch.zeros(1, t.numel() + 3, dtype=t.dtype, device="cuda")
        rows[:, :t.numel()] = t.detach().flatten()
        odd.append(rows.as_strided(t.shape, (t.numel() + 3, 64, 1)))
    odd[:3] = [t.detach().requires_grad_() for t in odd[:3]]
    assert all(torch.equal(a, b) for a, b in zip(run(*odd), want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_large_neighbours_change_no_rounding(cuda, dtype, d):
    """The next sequence's queries lie in this one's last tile; what they are changes no bit of this one's results."""
    lens = [300, 200]
    q, k, v, do = make(500, 4, 2, d, dtype, seed=6)
    with torch.no_grad():
        k[:300] *= torch.linspace(0.5, 2, 300, device="cuda")[:, None, None]      # (maxima that grow by less than 2^8)
    cu = on_device(bounds(lens))
    want = run(q, k, v, do, cu)
    with torch.no_grad():
        for t in (q, k, v, do):
            t[300:] *= 100
    for a, b in zip(run(q, k, v, do, cu), want):
        assert torch.equal(a[:300], b[:300])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_keys_ruled_out_by_infinities(cuda, dtype, d):
    """A document whose first keys are padding, ruled out by minus infinity in one place: whole tiles without a weight."""
    q, k, v, _ = make(400, 2, 1, d, dtype, seed=7)
    q, k, v = q.detach(), k.detach(), v.detach()
    q[..., 0], q[..., 1] = 1, 30
    k[:150, :, 0], k[150:, :, 0], k[150:, :, 1] = -float("inf"), 0, -30
    got = chb.causal_attention(q, k, v)
    want, tol = formula(q[150:], k[150:], v[150:], torch.zeros_like(q[150:]), [0, 250], d ** -0.5)
    assert ((got[150:].double() - want[0]).abs() <= tol[0]).all()
    assert got[:150].isnan().all()                               # (no key at all)


@pytest.mark.parametrize("h,hk,d,lens", [(2, 1, 128, [300, 2, 257]), (2, 2, 64, [640]), (3, 1, 40, [127, 0, 1, 128])])
def test_fp16_gradients_of_any_size(cuda, h, hk, d, lens):
    """Gradients are linear in dO, and a power of two rounds nothing: what 2^13 dO (whose dS is past fp16's largest value, while
    the results are not) and 2^-14 dO (whose dS is below its smallest one) give is that of dO times the power, but for the
    result's own rounding: half a step of both, or of 2^-24 below the normal range."""
    q, k, v, do = make(sum(lens), h, hk, d, torch.float16, seed=3)
    with torch.no_grad():
        q.mul_(0.25), k.mul_(0.25), v.mul_(4)
    do = in_eighths(do)
    cu = bounds(lens)
    want = check(q, k, v, do.half(), cu)
    for e in (13, -14):
        got = run(q, k, v, (do * 2.0 ** e).half(), on_device(cu))
        assert torch.equal(got[0], want[0])
        for a, b in zip(got[1:], want[1:]):
            # (a is off by 2^-11 |a| or 2^-25, the larger of them; b was, before its power: 2^-11 |b| or 2^-25 2^e)
            b = b.double() * 2.0 ** e
            assert ((a.double() - b).abs() <= 2.0 ** -10 * b.abs() + 2.0 ** -25 * (1 + 2.0 ** e)).all(), e


def test_fp16_gradients_of_sequences_of_different_size(cuda):
    """A sequence whose dO is 2^20 times another's changes nothing of the other's gradients, nor do rows that hold no number."""
    lens = [200, 300, 150]
    q, k, v, do = make(sum(lens), 4, 2, 64, torch.float16, seed=4)
    do = in_eighths(do)
    do[200:500] *= 2.0 ** 10
    do[:200] *= 2.0 ** -10
    do = do.half()
    cu = bounds(lens)
    got = run(q, k, v, do, on_device(cu))
    for s, e in zip(cu[:-1], cu[1:]):
        alone = run(*(t[s:e].detach().requires_grad_() for t in (q, k, v)), do[s:e])
        assert all(torch.equal(a[s:e], b) for a, b in zip(got[:2], alone))      # (dk and dv: heads may be shared out otherwise)
        want, tol = formula(*(t[s:e].detach() for t in (q, k, v)), do[s:e], [0, e - s], 0.125)
        size = do[s:e].abs().max().double() / 2                  # (the formula's tolerance is for dO of about 1)
        for a, b, t in zip(got, want, tol):
            assert ((a[s:e].double() - b).abs() <= t * max(size, 1.0) if s == 200 else (a[s:e].double() - b).abs() <= t).all()
    bad = do.clone()
    bad[250, 1, 3], bad[260, 0, 0] = float("nan"), float("inf")
    dq = run(q, k, v, bad, on_device(cu))[1]
    keep = torch.ones_like(dq, dtype=torch.bool)
    keep[250, 1] = keep[260, 0] = False
    assert torch.equal(dq[keep], got[1][keep]) and not dq[250, 1].isfinite().any()


def test_fp16_gradient_of_values_with_small_weights(cuda):
    """A key that every query behind it gives less than 2^-12: its dV is as exact, relative to its size, as any other's."""
    n, d = 1500, 64
    q, k, v, do = make(n, 1, 1, d, torch.float16, seed=5)
    with torch.no_grad():
        q[:, 0, 0], k[:, 0, 0], k[7, 0, 0] = 8, 0, -8            # (8 * -8 / 8 = -8: 2^-11.5 beside 2^-8 to 2^-11)
    dv = run(q, k, v, do, on_device([0, n]))[3]
    Q, K, G = (t.detach().double()[:, 0] for t in (q, k, do))
    keep = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    S = (Q @ K.t() / 8).masked_fill(~keep, -float("inf"))
    P = torch.softmax(S, -1)[100:, 7]                            # (of queries that see more than a hundred keys)
    full = torch.softmax(S, -1)[:, 7]
    assert P.max() < 2.0 ** -12
    E = 2.0 ** -24
    delta = 2 * d * E / 8 * (Q.abs() @ K.abs().t()).max() + 32 * E * (1 + S[keep].abs().max())
    size, want = full @ G.abs(), full @ G
    u = 2.0 ** -11
    assert ((dv[7, 0].double() - want).abs() <= (u + delta + (n + 16) * E) * size + u * want.abs() + 2.0 ** -25).all()


def test_fp16_captured_and_replayed_on_gradients_of_another_size(cuda):
    """The range is found on the device: a replay takes that of its own inputs."""
    q, k, v, do = make(400, 4, 2, 64, torch.float16, seed=9)
    do = in_eighths(do).half()
    cu = on_device([0, 150, 150, 390])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(chb.causal_attention(q, k, v, cu), (q, k, v), do)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:                                          # (two graphs of the same call share no workspace)
        with torch.cuda.graph(graph):
            outs.append(torch.autograd.grad(chb.causal_attention(q, k, v, cu), (q, k, v), do))
    for e in (2.0 ** 12, 2.0 ** -22):
        do *= e
        cu.copy_(on_device([0, 3, 300, 400]))
        for graph in graphs:
            graph.replay()
        want = run(q, k, v, do, cu)[1:]
        assert all(t.isfinite().all() and t.any() for t in want)
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_fp16_streams_at_once(cuda):
    inputs = [make(900, 4, 2, 64, torch.float16, seed=i) for i in range(2)]
    inputs[1][3].mul_(1000)
    cus = [on_device([0, 100, 900]), on_device([0, 33, 700, 890])]
    alone = [run(*inputs[i], cus[i]) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
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


def test_fp16_offsets_beyond_32_bits(cuda):
    T, h, d, n = (1 << 18) + 512, 64, 128, 512                # 2.15e9 elements of q and of dO
    g = torch.Generator(device="cuda").manual_seed(4)
    last = [torch.randn(n, x, d, generator=g, device="cuda").half() for x in (h, 1, 1, h)]
    last[3] *= 1000                                           # (the size of the last rows is theirs)
    big = [torch.zeros(T, x, d, dtype=torch.float16, device="cuda") for x in (h, 1, 1, h)]
    for b, t in zip(big, last):
        b[-n:] = t
    for t in big[:3] + last[:3]:
        t.requires_grad_()
    got = run(*big, on_device(list(range(0, T + 1, n))))
    alone = run(*last)
    assert all(torch.equal(a[-n:], b) for a, b in zip(got[:2], alone))
    # (dk and dv sum the heads in another order, as more CTAs share them: the formula's tolerance, n 2^-24 of the sum of sizes
    # among it, and not the other result's bits)
    want, tol = formula(*last, [0, n], d ** -0.5)
    for a, b, t in zip(got, want, tol):
        assert ((a[-n:].double() - b).abs() <= t).all() and not a[:-n].any()
