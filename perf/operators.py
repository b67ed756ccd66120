"""The operators of a decoder's training step, as cases to be timed and compared.

``attention``  causal attention over packed sequences with grouped heads; forward, or forward and gradients
``rotate``     norm of every query and key head and the position rotation, one pass; forward, or with gradients
``loss``       softmax cross entropy of a linear output layer; per-row losses, or the loss and its gradients

``run`` computes them in their plain form (32 bits, elementary operations, one rounding at the end) or, with ``own``
set, through this package.  ``exact`` computes them in 64 bits, each from its definition and apart from the plain form.
"""
import math

import torch

own = False

TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5                      # of the head norms
IGNORE = -100                   # label of a row that has no loss


def _attention(lens, heads, kv_heads, dim, dtype, train):
    """``lens``: lengths of the packed sequences, as text: "L" or "LxN" joined by commas."""
    return {"kind": "attention", "lens": lens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "train": train}


def _rotate(lens, heads, kv_heads, dim, dtype, train, norm=True, interleaved=True, first=0, base=10000.0):
    """``first``: position of every sequence's first token (a single token far in its text: a long one)."""
    return {"kind": "rotate", "lens": lens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "train": train, "norm": norm, "interleaved": interleaved, "first": first, "base": base}


def _loss(rows, dim, vocab, dtype, train, ignored=0.0, reduction="mean"):
    """``ignored``: share of the rows without a label."""
    return {"kind": "loss", "rows": rows, "dim": dim, "vocab": vocab, "dtype": dtype, "train": train, "ignored": ignored,
            "reduction": reduction}


def listed():
    cases = {
        # the tiny decoder's batch (2 x 32 tokens, 4 heads of 16) with an empty and a one-token sequence: latency counts
        "attention tiny": _attention("32x2,0,1,7", 4, 4, 16, "bf16", False),
        # a micro-batch of the GPT-2-medium shaped decoder, forward and backward
        "attention 8x1024 d64 train": _attention("1024x8", 16, 16, 64, "bf16", True),
        # a micro-batch of the 1.3B decoder, forward and backward
        "attention 4x2048 d128 train": _attention("2048x4", 16, 16, 128, "bf16", True),
        # documents of uneven length packed into one row of tokens, four query heads a key head
        "attention packed gqa fp16 train": _attention("1733,12,901,1,444,2048,77,1290,333,129,640,583", 16, 4, 128, "fp16", True),
        # one long prompt, forward only
        "attention 16384 gqa": _attention("16384", 16, 4, 128, "bf16", False),
        # queries and keys of a 1.3B decoder layer between projection and attention, forward and backward
        "rotate 4x2048 train": _rotate("2048x4", 16, 16, 128, "bf16", True),
        # one new token of each of 16 sequences, far in their texts
        "rotate 16 tokens": _rotate("1x16", 32, 8, 128, "fp16", False, interleaved=False, first=100003, base=500000.0),
        # packed documents, 32-bit activations, heads of 96, halves paired
        "rotate packed fp32 train": _rotate("1733,12,901,1,444,2048,77", 12, 4, 96, "fp32", True, interleaved=False),
        # the output layer of the GPT-2-medium shaped decoder: every token of a micro-batch
        "loss 8192x1024x50257 train": _loss(8192, 1024, 50257, "bf16", True),
        # the output layer of the 1.3B decoder
        "loss 8192x2048x32000 train": _loss(8192, 2048, 32000, "bf16", True),
        # the score of a short completion: a loss for each token, no gradients
        "loss 33 rows": _loss(33, 1024, 50257, "bf16", False, reduction="none"),
        # a fine-tuning batch whose prompt tokens have no label, sizes that no tile divides
        "loss odd fp16 train": _loss(1001, 520, 10007, "fp16", True, ignored=0.4, reduction="sum"),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_lens(rng, most):
    total, n = _log(rng, 1, most), _log(rng, 1, 24)
    if rng.random() < 0.3:
        return "%dx%d" % (max(1, total // n), n)
    cuts = sorted(rng.randrange(total + 1) for _ in range(n - 1))        # empty sequences among them
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng):
    kind = rng.choice(("attention", "attention", "rotate", "loss"))
    kv = rng.choice((1, 2, 3, 4, 5, 8))
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 7, 8) if kv * g <= 16])
    if kind == "attention":
        train = rng.random() < 0.6
        dim = rng.choice((64, 128, 64, 128, 64, 128, 16, 32, 40, 80, 96, 112))
        return _attention(_draw_lens(rng, 6144 if train else 16384), heads, kv, dim, rng.choice(("bf16", "bf16", "fp16")), train)
    if kind == "rotate":
        return _rotate(_draw_lens(rng, 8192), heads, kv, rng.choice((16, 32, 64, 64, 96, 128, 128, 192, 256)),
                       rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.6, rng.random() < 0.7,
                       rng.random() < 0.5, rng.choice((0, 0, _log(rng, 1, 1 << 20))), rng.choice((10000.0, 500000.0)))
    dim, vocab = 8 * _log(rng, 8, 256), _log(rng, 100, 64000)
    rows = _log(rng, 1, max(1, min(16384, 8192 * 2048 * 32000 // (dim * vocab))))
    return _loss(rows, dim, vocab, rng.choice(("bf16", "bf16", "fp16")), rng.random() < 0.7, rng.choice((0.0, 0.1, 0.6)),
                 rng.choice(("mean", "mean", "sum", "none")))


def _lens(case):
    parts = [p.split("x") for p in case["lens"].split(",")]
    return [int(p[0]) for p in parts for _ in range(int(p[1]) if len(p) > 1 else 1)]


def _bounds(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def prepare(case, seed):
    dev, dt = "cuda", TYPE[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev)      # noqa: E731
    train = case["train"]
    state = {"case": case}
    leaf = lambda t: t.to(dt).requires_grad_(train)                 # noqa: E731
    if case["kind"] == "loss":
        n, d, v = case["rows"], case["dim"], case["vocab"]
        targets = torch.randint(0, v, (n,), generator=g, device=dev)
        weight = (rand(v, d) * (1.6 / math.sqrt(d))).to(dt)         # logits of standard deviation 1.6 ...
        x = rand(n, d) + 0.8 * weight[targets].float()              # ... and somewhat more at the label
        if case["ignored"]:
            targets = torch.where(torch.rand(n, generator=g, device=dev) < case["ignored"], IGNORE, targets)
            targets[n // 2] = v // 2                                # (a mean has a row at least)
        state.update(x=leaf(x), weight=leaf(weight), targets=targets)
        if train:
            state["grad"] = rand(n) if case["reduction"] == "none" else torch.full((), 1.5, device=dev)
        return state
    lens = _lens(case)
    cu = _bounds(lens)
    T, h, hk, dim = cu[-1], case["heads"], case["kv_heads"], case["dim"]
    state.update(lens=lens, cu=torch.tensor(cu, dtype=torch.int32, device=dev))
    if case["kind"] == "attention":
        state.update(q=leaf(rand(T, h, dim)), k=leaf(rand(T, hk, dim)), v=leaf(rand(T, hk, dim)))
        if train:
            state["do"] = rand(T, h, dim).to(dt)
        return state
    pos = [case["first"] + i for n in lens for i in range(n)]
    # queries and keys as a projection leaves them: heads of uneven size, some values far out
    state.update(q=leaf(rand(T, h, dim) * (0.5 + 2 * torch.rand(1, h, 1, generator=g, device=dev))),
                 k=leaf(rand(T, hk, dim) * (0.5 + 2 * torch.rand(1, hk, 1, generator=g, device=dev))),
                 positions=torch.tensor(pos, dtype=torch.int32, device=dev), wq=None, wk=None)
    if case["norm"]:
        state.update(wq=leaf(1 + 0.2 * rand(dim)), wk=leaf(1 + 0.2 * rand(dim)))
    if train:
        state.update(dq=rand(T, h, dim).to(dt), dk=rand(T, hk, dim).to(dt))
    return state


# ---------------------------------------------------------------------------------------------------- plain forms

def _plain_attention(q, k, v, lens):
    group, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    parts = []
    for qs, ks, vs in zip(*(t.float().transpose(0, 1).split(lens, dim=1) for t in (q, k, v))):      # one sequence
        n = qs.shape[1]
        s = torch.matmul(qs.reshape(ks.shape[0], group * n, ks.shape[2]), ks.transpose(1, 2)).view(q.shape[1], n, n) * scale
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=s.device).triu(1), -math.inf)
        if n:
            s = torch.exp(s - s.amax(-1, keepdim=True))
        p = s / s.sum(-1, keepdim=True)
        parts.append(torch.matmul(p.view(ks.shape[0], group * n, n), vs).view(qs.shape))
    return torch.cat(parts, dim=1).transpose(0, 1).to(q.dtype)


def _plain_rotate(x, weight, positions, interleaved, base):
    y, d = x.float(), x.shape[-1]
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    freq = base ** (-torch.arange(0, d, 2, device=x.device, dtype=torch.float64) / d)
    angle = positions.double()[:, None, None] * freq                # (64 bits: positions may be far)
    cos, sin = angle.cos().float(), angle.sin().float()
    a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :d // 2], y[..., d // 2:])
    c, e = a * cos - b * sin, a * sin + b * cos
    return (torch.stack((c, e), -1).flatten(-2) if interleaved else torch.cat((c, e), -1)).to(x.dtype)


def _plain_loss(x, weight, targets, reduction):
    logits = torch.matmul(x.float(), weight.float().t())
    top = logits.detach().amax(-1, keepdim=True)
    lse = torch.log(torch.exp(logits - top).sum(-1)) + top[:, 0]
    valid = targets != IGNORE
    at = logits.gather(1, targets.clamp(min=0)[:, None])[:, 0]
    rows = torch.where(valid, lse - at, torch.zeros_like(lse))
    return rows if reduction == "none" else rows.sum() / valid.sum() if reduction == "mean" else rows.sum()


def run(state):
    case, train = state["case"], state["case"]["train"]
    if own:
        import configurable_hierarchical_allreduce_algorithms_b200 as chb
    if case["kind"] == "attention":
        q, k, v = state["q"], state["k"], state["v"]
        if own:
            o = chb.causal_attention(q, k, v, state["cu"])
        else:
            o = _plain_attention(q, k, v, state["lens"])
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), state["do"])) if train else o
    if case["kind"] == "rotate":
        q, k, wq, wk = state["q"], state["k"], state["wq"], state["wk"]
        if own:
            a, b = chb.head_norm_rope(q, k, wq, wk, state["positions"], eps=EPS, base=case["base"], interleaved=case["interleaved"])
        else:
            a = _plain_rotate(q, wq, state["positions"], case["interleaved"], case["base"])
            b = _plain_rotate(k, wk, state["positions"], case["interleaved"], case["base"])
        if not train:
            return a, b
        leaves = (q, k) if wq is None else (q, k, wq, wk)
        return (a.detach(), b.detach(), *torch.autograd.grad((a, b), leaves, (state["dq"], state["dk"])))
    x, weight = state["x"], state["weight"]
    if own:
        loss = chb.linear_cross_entropy(x, weight, state["targets"], ignore_index=IGNORE, reduction=case["reduction"])
    else:
        loss = _plain_loss(x, weight, state["targets"], case["reduction"])
    return (loss.detach(), *torch.autograd.grad(loss, (x, weight), state["grad"])) if train else loss


# ---------------------------------------------------------------------------------------------- floors and 64 bits

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "loss":
        n, d, v = case["rows"], case["dim"], case["vocab"]
        both = (n + v) * d * size
        return {"bytes": both * (2 if case["train"] else 1) + 8 * n, "flops": 2 * n * d * v * (3 if case["train"] else 1)}
    lens = _lens(case)
    T, h, hk, dim = sum(lens), case["heads"], case["kv_heads"], case["dim"]
    q, k = T * h * dim * size, T * hk * dim * size
    if case["kind"] == "attention":
        pairs = sum(n * (n + 1) // 2 for n in lens)
        # forward q, k, v -> o; backward with do -> dq, dk, dv; two products forward, five backward
        return {"bytes": 2 * q + 2 * k + (2 * q + 2 * k if case["train"] else 0), "flops": 2 * pairs * h * dim * (7 if case["train"] else 2)}
    return {"bytes": (2 if not case["train"] else 4) * (q + k) + 4 * T, "flops": 10 * T * (h + hk) * dim * (3 if case["train"] else 1)}


def _exact_attention(state):
    case = state["case"]
    q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    outs = [torch.zeros_like(t) for t in ((q, q, k, v) if case["train"] else (q,))]
    cu = _bounds(state["lens"])
    for s, e in zip(cu[:-1], cu[1:]):
        for h in range(case["heads"]):
            kk, vv = k[s:e, h // group], v[s:e, h // group]
            for r in range(s, e, 2048):                         # rows of queries: they see the keys up to their own
                z = min(e, r + 2048)
                scores = (q[r:z, h] @ kk[:z - s].t()) * scale
                rows, cols = torch.arange(r, z, device=q.device)[:, None], torch.arange(s, z, device=q.device)[None]
                scores[cols > rows] = -math.inf
                p = (scores - torch.logsumexp(scores, 1, keepdim=True)).exp()
                o = p @ vv[:z - s]
                outs[0][r:z, h] = o
                if case["train"]:
                    do = state["do"][r:z, h].double()
                    ds = p * (do @ vv[:z - s].t() - (do * o).sum(1, keepdim=True)) * scale
                    outs[1][r:z, h] = ds @ kk[:z - s]
                    outs[2][s:z, h // group] += ds.t() @ q[r:z, h]
                    outs[3][s:z, h // group] += p.t() @ do
    return tuple(outs) if case["train"] else outs[0]


def _exact_rotate(state):
    case, outs, grads, weights = state["case"], [], [], []
    d = case["dim"]
    i = torch.arange(d // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + d // 2)
    angle = torch.outer(state["positions"].double(), torch.exp(-2.0 * i.double() / d * math.log(case["base"])))[:, None]
    for name, wname, dname in (("q", "wq", "dq"), ("k", "wk", "dk")):
        x = state[name].detach().double()
        w = torch.ones(d, dtype=torch.float64, device="cuda") if state[wname] is None else state[wname].detach().double()
        inv = 1.0 / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS) if case["norm"] else torch.ones_like(x[..., :1])
        turn = torch.polar(torch.ones_like(angle), angle)
        z = torch.complex((x * inv * w)[..., first], (x * inv * w)[..., second]) * turn
        y = torch.empty_like(x)
        y[..., first], y[..., second] = z.real, z.imag
        outs.append(y)
        if not case["train"]:
            continue
        gy = state[dname].double()
        z = torch.complex(gy[..., first], gy[..., second]) * turn.conj()
        u = torch.empty_like(x)
        u[..., first], u[..., second] = z.real, z.imag
        weights.append((u * x * inv).sum((0, 1)))
        u = u * w
        grads.append(inv * (u - x * inv.pow(2) * (u * x).mean(-1, keepdim=True)) if case["norm"] else u)
    return tuple(outs + grads + (weights if case["norm"] else []))


def _exact_loss(state):
    case = state["case"]
    x, w, targets = state["x"].detach().double(), state["weight"].detach().double(), state["targets"]
    valid = targets != IGNORE
    rows = torch.zeros(len(x), dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    each = 1.0 / int(valid.sum()) if case["reduction"] == "mean" else 1.0
    for part in valid.nonzero()[:, 0].split(2048):
        logp = torch.log_softmax(x[part] @ w.t(), 1)
        at = torch.arange(len(part), device="cuda"), targets[part]
        rows[part] = -logp[at]
        if case["train"]:
            p = logp.exp()
            p[at] -= 1.0
            p *= (state["grad"][part, None] if case["reduction"] == "none" else state["grad"] * each).double()
            dx[part] = p @ w
            dw += p.t() @ x[part]
    loss = rows if case["reduction"] == "none" else rows.sum() * each
    return (loss, dx, dw) if case["train"] else loss


def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": _exact_attention, "rotate": _exact_rotate, "loss": _exact_loss}[case["kind"]](state)
