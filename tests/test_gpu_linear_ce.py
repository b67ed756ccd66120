"""Cross entropy of a linear output layer against the formula in 64 bits, loss and gradients.

Tolerances, element by element, with u = half a step of the operands' type (eps / 2) and e = 2^-24:
a logit is a sum of D exact products in fp32, off by at most delta = D e sum|x||w| (largest over the vocabulary); a
probability by a factor 1 + 2 delta (its own logit and the normaliser) + 16 e (exponential, logarithm, weights);
dx = G W sums V products of a G rounded once: (u + 2 delta + (V + 16) e) |P + onehot| g |W|, and one rounding of the
result, u |dx|; dW alike with the rows summed.  fp16 keeps G times 2^14 relative to the largest g: a G below fp16's
normal range is off by up to 2^-25 2^-14 max|g| instead."""
import pytest
import torch

import configurable_hierarchical_allreduce_algorithms_b200 as chb

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def formula(x, w, t, g, ignore, reduction):
    """Loss, gradients and their tolerances in 64 bits; g: gradient of the loss."""
    u = torch.finfo(x.dtype).eps / 2
    small = 2.0 ** -39 if x.dtype == torch.float16 else 0.0
    x, w = x.detach().double(), w.detach().double()
    keep = (t != ignore).nonzero()[:, 0]
    xs, ts = x[keep], t[keep]
    logp = torch.log_softmax(xs @ w.t(), -1)
    rows = torch.zeros(len(x), dtype=torch.float64, device=x.device)
    at = torch.arange(len(keep), device=x.device), ts
    rows[keep] = -logp[at]
    n, (v, d) = max(1, len(keep)), w.shape
    loss = rows if reduction == "none" else rows.sum() / (len(keep) if reduction == "mean" else 1)
    delta = d * E * (xs.abs() @ w.abs().t()).amax(-1, keepdim=True) if len(keep) else torch.zeros(0, 1, device=x.device)
    tol_rows = torch.zeros_like(rows)
    tol_rows[keep] = 2 * delta[:, 0] + 16 * E * (1 + logp.abs().amax(-1) if len(keep) else 0)
    tol = tol_rows if reduction == "none" else tol_rows.sum() / (n if reduction == "mean" else 1) + 4 * E * loss.abs()
    gr = (g[keep] if reduction == "none" else (g / n if reduction == "mean" else g).expand(len(keep))).double()[:, None]
    p = logp.exp()
    size = p.clone()
    p[at] -= 1
    size[at] += 1
    G, top = p * gr, gr.abs().max() if len(keep) else 0.0
    size = size * gr.abs()
    rel = u + 2 * delta
    dx, tdx = torch.zeros_like(x), torch.zeros_like(x)
    dx[keep] = G @ w
    tdx[keep] = (size * (rel + (v + 16) * E) + small * top) @ w.abs() + u * dx[keep].abs()
    dw = G.t() @ xs
    tdw = (size * (rel + (n + 16) * E) + small * top).t() @ xs.abs() + u * dw.abs()
    tiny = 2.0 ** -25 if small else 0.0      # (results below fp16's normal range)
    return loss, dx, dw, tol, tdx + tiny, tdw + tiny


def make(n, d, v, dtype, ignored=0.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, d, generator=g, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(v, d, generator=g, device="cuda") * (1.6 / d ** 0.5)).to(dtype).requires_grad_()
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    if ignored:
        t[torch.rand(n, generator=g, device="cuda") < ignored] = -100
    return x, w, t


def check(x, w, t, reduction, grad=None, ignore=-100):
    if grad is None:
        g = torch.Generator(device="cuda").manual_seed(9)
        grad = torch.randn(len(x), generator=g, device="cuda") if reduction == "none" else torch.tensor(1.5, device="cuda")
    loss = chb.linear_cross_entropy(x, w, t, reduction=reduction, ignore_index=ignore)
    dx, dw = torch.autograd.grad(loss, (x, w), grad)
    chb.check_operators()
    want = formula(x, w, t, grad, ignore, reduction)
    for got, ref, tol in zip((loss, dx, dw), want[:3], want[3:]):
        assert got.shape == ref.shape
        assert ((got.double() - ref).abs() <= tol).all(), ((got.double() - ref).abs() - tol).max()
    return loss, dx, dw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("n,d,v,ignored", [(1, 8, 1, 0), (1, 64, 257, 0), (127, 72, 255, 0.5), (128, 64, 256, 0),
                                           (129, 136, 513, 0.3), (700, 520, 1009, 0.6), (257, 1024, 4100, 0.1)])
def test_matches_the_formula(cuda, dtype, reduction, n, d, v, ignored):
    check(*make(n, d, v, dtype, ignored, seed=n + d), reduction)


def test_several_pieces_of_the_vocabulary(cuda):
    check(*make(8192, 64, 7001, torch.bfloat16, 0.2), "mean")      # 114 MB of G


def test_more_pieces_of_the_vocabulary(cuda):
    check(*make(9000, 72, 25001, torch.float16, 0.05), "mean")     # more than 400 MB of G: three pieces of 192 MiB


def test_negative_and_zero_gradients(cuda):
    x, w, t = make(200, 64, 300, torch.float16)
    check(x, w, t, "mean", torch.tensor(-2.0, device="cuda"))
    check(x, w, t, "none", torch.where(torch.arange(200, device="cuda") % 3 == 0, 0.0, -1.0))
    for reduction, g in (("sum", torch.zeros((), device="cuda")), ("none", torch.zeros(200, device="cuda"))):
        loss = chb.linear_cross_entropy(x, w, t, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (x, w), g)
        assert not dx.any() and not dw.any()


def test_rows_without_a_label_reach_nothing(cuda):
    x, w, t = make(300, 128, 515, torch.bfloat16, 0.4)
    a = check(x, w, t, "mean")
    bad = x.detach().clone()
    out = (t == -100).nonzero()[:, 0]
    bad[out[0::2]] = float("nan")
    bad[out[1::2]] = float("inf")
    bad.requires_grad_()
    loss = chb.linear_cross_entropy(bad, w, t)
    b = (loss, *torch.autograd.grad(loss, (bad, w), torch.tensor(1.5, device="cuda")))
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    assert not b[1][out].any()


def test_no_row_has_a_label(cuda):
    x, w, t = make(130, 64, 300, torch.bfloat16)
    t[:] = 7
    for reduction in ("none", "mean", "sum"):
        loss = chb.linear_cross_entropy(x, w, t, ignore_index=7, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
        assert loss.isnan().all() if reduction == "mean" else not loss.any()
        assert not dx.any() and not dw.any()


def test_a_label_outside_the_vocabulary_makes_its_row_nan(cuda):
    x, w, t = make(64, 64, 300, torch.bfloat16)
    t[5], t[9] = 300, -1
    loss = chb.linear_cross_entropy(x, w, t, reduction="none")
    assert loss.isnan().nonzero()[:, 0].tolist() == [5, 9]
    assert chb.linear_cross_entropy(x, w, t).isnan()


def test_large_logits_and_infinite_ones(cuda):
    x, w, t = make(100, 64, 300, torch.bfloat16)
    x = (x.detach() * 40).requires_grad_()                        # logits of hundreds: all but one exponential vanish
    check(x, w, t, "none")
    w2 = w.detach().clone()
    w2[17, 0] = -float("inf")                                     # a token that is ruled out where x's first value is positive
    x2 = x.detach().clone()
    x2[:, 0] = x2[:, 0].abs() + 1
    t = torch.where(t == 17, 18, t)
    loss = chb.linear_cross_entropy(x2, w2, t, reduction="none")
    ref = torch.nn.functional.cross_entropy(x2.double() @ w2.double().t(), t, reduction="none")
    assert loss.isfinite().all() and torch.allclose(loss.double(), ref, rtol=1e-5, atol=1e-3)      # (64 * 2^-24 * sum|x||w| < 1e-3)


def test_strided_unaligned_and_shaped_inputs(cuda):
    x, w, t = make(96, 72, 300, torch.bfloat16)
    want = chb.linear_cross_entropy(x, w, t, reduction="none")
    wide = torch.zeros(96, 2 * 72 + 1, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:73] = x.detach()
    assert torch.equal(chb.linear_cross_entropy(wide[:, 1:73], w, t, reduction="none"), want)
    tall = w.detach().t().contiguous().t()
    assert torch.equal(chb.linear_cross_entropy(x, tall, t, reduction="none"), want)
    shaped = chb.linear_cross_entropy(x.view(4, 24, 72), w, t.view(4, 24), reduction="none")
    assert shaped.shape == (4, 24) and torch.equal(shaped.flatten(), want)
    dx, = torch.autograd.grad(shaped.sum(), x)                     # (an expanded gradient)
    assert dx.shape == x.shape
    one = chb.linear_cross_entropy(x[3], w, t[3])
    assert one.shape == () and torch.equal(one, want[3])


def test_one_gradient_only_and_repeatable(cuda):
    x, w, t = make(500, 128, 1000, torch.bfloat16, 0.2)
    loss = chb.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    for _ in range(3):
        again = chb.linear_cross_entropy(x, w, t)
        assert torch.equal(again, loss)
        assert torch.equal(torch.autograd.grad(again, x, retain_graph=True)[0], dx)
        assert torch.equal(torch.autograd.grad(again, w)[0], dw)
    only_x = chb.linear_cross_entropy(x, w.detach(), t)
    assert torch.equal(torch.autograd.grad(only_x, x)[0], dx)


def test_no_rows(cuda):
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = torch.zeros(10, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert chb.linear_cross_entropy(x, w, t).isnan()
    assert chb.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
    w.data[0, 0] = float("inf")
    s = chb.linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(s, (x, w))
    assert s == 0 and dx.shape == x.shape and not dw.any()


def test_differences(cuda):
    """The gradient against differences of the loss along a direction (fp16 steps that the type holds exactly)."""
    x, w, t = make(40, 64, 200, torch.float16)
    loss = chb.linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    for leaf, grad in ((x, dx), (w, dw)):
        g = torch.Generator(device="cuda").manual_seed(3)
        step = torch.randint(-1, 2, leaf.shape, generator=g, device="cuda").double() * 2.0 ** -6
        at = [(leaf.detach().double() + s * step).to(torch.float16) for s in (1, -1)]
        real = (at[0].double() - at[1].double())                   # (what is left of the steps after rounding)
        f = [chb.linear_cross_entropy(a if leaf is x else x, a if leaf is w else w, t, reduction="sum").double() for a in at]
        slope = (real * grad.double()).sum()
        # second order cancels; third order: |step x w|^3 ~ (64 * 2^-6 * 0.2)^3 / 6 a row at the very most
        assert abs(f[0] - f[1] - slope) <= 0.02 * abs(slope) + 40 * 0.2 ** 3 / 3


def test_captured_and_replayed_on_new_inputs(cuda):
    x, w, t = make(300, 128, 1000, torch.bfloat16, 0.3)
    grad = torch.tensor(1.0, device="cuda")

    def step():
        loss = chb.linear_cross_entropy(x, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w), grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    x2, w2, t2 = make(300, 128, 1000, torch.bfloat16, 0.7, seed=5)
    with torch.no_grad():
        x.copy_(x2), w.copy_(w2), t.copy_(t2)
    graph.replay()
    for a, b in zip(outs, step()):
        assert torch.equal(a, b)


def test_offsets_beyond_32_bits(cuda):
    n, d, v, last = 66000, 32768, 96, 40                       # 2.16e9 elements of x
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.zeros(n, d, dtype=torch.bfloat16, device="cuda")
    x[-last:] = torch.randn(last, d, generator=g, device="cuda").bfloat16()
    w = (torch.randn(v, d, generator=g, device="cuda") * (1.6 / d ** 0.5)).bfloat16().requires_grad_()
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    grad = torch.zeros(n, device="cuda")
    grad[-last:] = torch.randn(last, generator=g, device="cuda")
    x.requires_grad_()
    loss = chb.linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, (x, w), grad)
    want = formula(x[-last:], w, t[-last:], grad[-last:], -100, "none")
    for got, ref, tol in zip((loss[-last:], dx[-last:], dw), want[:3], want[3:]):
        # (dw is summed over all rows: 66000 more terms of zero add nothing)
        assert ((got.double() - ref).abs() <= tol).all(), ((got.double() - ref).abs() - tol).max()
    assert not dx[:-last].any()


def test_two_streams_at_once(cuda):
    """Calls that overlap share nothing: each stream's results are those of the call alone."""
    inputs = [make(700, 256, 3000, torch.bfloat16, 0.3, seed=i) for i in range(2)]
    grad = torch.ones((), device="cuda")

    def step(i):
        x, w, t = inputs[i]
        loss = chb.linear_cross_entropy(x, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w), grad))

    alone = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, alone[i]))
    chb.check_operators()
