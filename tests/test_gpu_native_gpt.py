"""The decoder with its attention, rotation and loss on this library's kernels: the operators in one model, as a training
step uses them.  Both sides round activations to bf16 after every operator; the kernels round no more often than torch's
operators do, so the whole gradient may be off the 64-bit one by what torch's bf16 model is off, and half as much again."""
import copy
import dataclasses
import json

import pytest
import torch

from configurable_hierarchical_allreduce_algorithms_b200.models.gpt import GPT, GPTConfig

pytestmark = pytest.mark.gpu


def gradients(model, idx, targets, cu):
    model.zero_grad()
    loss = model(idx, targets, cu_seqlens=cu)
    loss.backward()
    return loss.detach().double(), torch.cat([p.grad.double().flatten() for p in model.parameters()])


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("style,kw", [("gpt2", {}), ("llama", {}), ("gpt2", {"n_kv_head": 2}), ("llama", {"n_kv_head": 1, "qk_norm": True})])
def test_as_exact_as_torch(cuda, style, kw, packed):
    torch.manual_seed(0)
    cfg = dataclasses.replace(GPTConfig.tiny(style), **kw)
    plain = GPT(cfg).cuda().bfloat16()
    native = copy.deepcopy(plain)
    for m in [native, *native.blocks]:
        m.cfg = dataclasses.replace(cfg, native=True)
    exact = copy.deepcopy(plain).double()
    idx = torch.randint(0, 257, (4, 32), device="cuda")
    targets = torch.where(torch.rand(idx.shape, device="cuda") < 0.2, -100, idx.roll(-1, 1))
    cu = torch.tensor([0, 3, 3, 33, 34, 64, 96, 97, 128], dtype=torch.int32, device="cuda") if packed else None
    loss, want = gradients(exact, idx, targets, cu)
    off = []
    for m in (plain, native):
        a, g = gradients(m, idx, targets, cu)
        off.append((abs(a - loss), (g - want).norm()))
    assert off[1][1] <= 1.5 * off[0][1]
    assert off[1][0] <= 1.5 * off[0][0] + 2.0 ** -9 * loss
    logits = native(idx, cu_seqlens=cu)
    assert logits.shape == (4, 32, 257)


@pytest.mark.parametrize("mode", ["dp", "zero"])
def test_training_command(cuda, mode, capsys):
    from configurable_hierarchical_allreduce_algorithms_b200.bench import train

    train.main(["--mode", mode, "--tiny", "--native", "--steps", "2", "--warmup", "1"])
    out = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert out["native"] and out["loss"] == out["loss"]
