"""The decoder operators and what torch can do around a call: forward-mode derivatives, a first call inside a capture,
batches without tokens."""
import subprocess
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import configurable_hierarchical_allreduce_algorithms_b200 as chb
from configurable_hierarchical_allreduce_algorithms_b200.models.gpt import GPT, GPTConfig

pytestmark = pytest.mark.gpu


def calls():
    r = lambda *s: torch.randn(*s, device="cuda").bfloat16()      # noqa: E731
    q, k, v, x, w = r(9, 2, 16), r(9, 1, 16), r(9, 1, 16), r(9, 16), r(20, 16)
    t = torch.arange(9, device="cuda")
    return {"attention": (chb.causal_attention, (q, k, v)), "rotate": (chb.head_norm_rope, (q, k)),
            "loss": (lambda x, w: chb.linear_cross_entropy(x, w, t), (x, w))}


@pytest.mark.parametrize("name", ["attention", "rotate", "loss"])
def test_forward_mode_is_refused(cuda, name):
    """A tangent is never dropped: no result may look like a constant."""
    fn, args = calls()[name]
    plain = fn(*args)
    with fwAD.dual_level():
        for n in range(len(args)):
            dual = [fwAD.make_dual(a, torch.ones_like(a)) if i == n else a for i, a in enumerate(args)]
            with pytest.raises((NotImplementedError, RuntimeError), match="(?i)forward"):
                fn(*dual)
        again = fn(*args)                                          # (no tangent: an ordinary call)
    for a, b in zip(plain if name == "rotate" else (plain,), again if name == "rotate" else (again,)):
        assert torch.equal(a, b)
    leaf = args[0].detach().requires_grad_()
    out = fn(leaf, *args[1:])
    out = out[0] if name == "rotate" else out
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="forward"):
        torch.autograd.grad(out, leaf, fwAD.make_dual(torch.ones_like(out), torch.ones_like(out)))
    with pytest.raises(Exception):
        torch.func.jvp(fn, args, tuple(torch.ones_like(a) for a in args))


FIRST = """
import torch, configurable_hierarchical_allreduce_algorithms_b200 as chb
r = lambda *s: torch.randn(*s, device="cuda").bfloat16().requires_grad_()
q, k, v, x, w = r(300, 4, 64), r(300, 2, 64), r(300, 2, 64), r(300, 64), r(500, 64)
t, one = torch.arange(300, device="cuda"), torch.ones((), device="cuda")
do = torch.randn(300, 4, 64, device="cuda").bfloat16()
def step():
    a, b = chb.head_norm_rope(q, k)
    o = chb.causal_attention(a, b, v)
    loss = chb.linear_cross_entropy(x, w, t)
    return (o.detach(), loss.detach(), *torch.autograd.grad(o, (q, k, v), do), *torch.autograd.grad(loss, (x, w), one))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outs, step()))
print("captured")
"""


def test_first_calls_inside_a_capture(cuda):
    r = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("shape", [(2, 0), (0, 8), (0, 0)])
@pytest.mark.parametrize("style", ["gpt2", "llama"])
def test_batches_without_tokens(cuda, style, shape):
    cfg = GPTConfig.tiny(style)
    cfg.native = True
    model = GPT(cfg).cuda().bfloat16()
    idx = torch.zeros(shape, dtype=torch.long, device="cuda")
    assert model(idx).shape == (*shape, cfg.vocab)
    loss = model(idx, idx)
    loss.backward()
    assert loss.isnan()
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert model(idx, cu_seqlens=cu).shape == (*shape, cfg.vocab)
