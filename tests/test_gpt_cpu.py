"""The decoder's variants on the CPU: shared key heads, head norms, packed documents."""
import dataclasses

import pytest
import torch

from configurable_hierarchical_allreduce_algorithms_b200.models.gpt import GPT, GPTConfig


def tiny(style, **kw):
    torch.manual_seed(0)
    return GPT(dataclasses.replace(GPTConfig.tiny(style), **kw)).double()


@pytest.mark.parametrize("style,kw", [("gpt2", {}), ("llama", {}), ("gpt2", {"n_kv_head": 2}), ("llama", {"n_kv_head": 1, "qk_norm": True})])
def test_packed_documents_are_documents(style, kw):
    m = tiny(style, **kw)
    idx = torch.randint(0, 257, (2, 32))
    flat, cu = idx.view(-1), [0, 5, 5, 31, 40, 64]            # (documents may run over the end of a row)
    got = m(idx, cu_seqlens=torch.tensor(cu, dtype=torch.int32)).view(64, -1)
    for s, e in zip(cu[:-1], cu[1:]):
        if e > s:
            want = m(flat[None, s:e])[0]
            assert (got[s:e] - want).abs().max() <= 1e-9 * want.abs().max()


def test_rows_are_documents_without_bounds():
    m = tiny("llama", n_kv_head=2, qk_norm=True)
    idx = torch.randint(0, 257, (2, 32))
    loss = m(idx, idx)
    packed = m(idx, idx, cu_seqlens=torch.tensor([0, 32, 64], dtype=torch.int32))
    assert abs(loss - packed) <= 1e-9 * abs(loss)


def test_shared_key_heads_are_repeated_ones():
    few, many = tiny("llama", n_kv_head=2), tiny("llama")      # (heads of 16: 64 rows of queries, 32 of keys, 32 of values)
    state = few.state_dict()
    for n, w in list(state.items()):
        if n.endswith("qkv.weight"):
            q, k, v = w.split([64, 32, 32])
            state[n] = torch.cat([q, *(t.view(2, 16, 64).repeat_interleave(2, 0).reshape(64, 64) for t in (k, v))])
    many.load_state_dict(state)
    idx = torch.randint(0, 257, (2, 32))
    a, b = few(idx), many(idx)
    assert (a - b).abs().max() <= 1e-9 * b.abs().max()
