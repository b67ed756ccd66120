"""Decoder-only transformers used by the data-parallel and sharded-optimizer
paths: a GPT-2 style block (LayerNorm, GELU MLP, learned positions) and a
Llama style block (RMSNorm, SwiGLU, rotary positions).  GEMMs go to the vendor
libraries through PyTorch; this library's kernels are the collectives and the
fused optimizer / gradient steps around them and, with ``native=True`` (bf16 or
fp16 parameters on a GPU), causal attention, the head norm with the rotation, and
the loss of the output layer (``ops/decoder.py``).  A program that runs these
asks ``check_operators()`` before it uses a result or writes a checkpoint, as it
asks the communicator: both synchronise."""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import decoder


@dataclass
class GPTConfig:
    n_layer: int = 24
    d_model: int = 1024
    n_head: int = 16
    vocab: int = 50257
    seq_len: int = 1024
    ffn: int = 0            # 0: 4 * d_model (GPT-2); Llama style uses an explicit SwiGLU width
    style: str = "gpt2"     # "gpt2" | "llama"
    n_kv_head: int = 0      # key / value heads, each shared by n_head / n_kv_head query heads; 0: n_head
    qk_norm: bool = False   # RMS norm of every query and key head before the rotation (llama style)
    native: bool = False    # attention, rotation and loss on this library's kernels

    @staticmethod
    def gpt2_medium():
        return GPTConfig(24, 1024, 16, 50257, 1024, 0, "gpt2")

    @staticmethod
    def llama_1p3b():
        return GPTConfig(24, 2048, 16, 32000, 2048, 5504, "llama")

    @staticmethod
    def tiny(style="gpt2"):
        return GPTConfig(2, 64, 4, 257, 32, 0 if style == "gpt2" else 176, style)


class RMSNorm(nn.Module):
    def __init__(self, d, eps=1e-5):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d))
        self.eps = eps

    def forward(self, x):
        return F.rms_norm(x, (x.shape[-1],), self.weight, self.eps)


def _rope(q, k, base=10000.0, pos=None):
    # q, k: [B, H, T, D]; pos: [B, T], or None: 0, 1, 2, ...
    T, D = q.shape[-2], q.shape[-1]
    inv = 1.0 / (base ** (torch.arange(0, D, 2, device=q.device, dtype=torch.float32) / D))
    if pos is None:
        ang = torch.outer(torch.arange(T, device=q.device, dtype=torch.float32), inv)
    else:
        ang = pos.to(torch.float32)[:, None, :, None] * inv
    cos, sin = ang.cos().to(q.dtype), ang.sin().to(q.dtype)

    def rot(x):
        x1, x2 = x[..., 0::2], x[..., 1::2]
        return torch.stack((x1 * cos - x2 * sin, x1 * sin + x2 * cos), dim=-1).flatten(-2)

    return rot(q), rot(k)


class Block(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        d = cfg.d_model
        self.cfg = cfg
        llama = cfg.style == "llama"
        self.ln1 = RMSNorm(d) if llama else nn.LayerNorm(d)
        self.ln2 = RMSNorm(d) if llama else nn.LayerNorm(d)
        self.hd, self.kv = d // cfg.n_head, cfg.n_kv_head or cfg.n_head
        self.qkv = nn.Linear(d, d + 2 * self.kv * self.hd, bias=not llama)
        self.q_norm, self.k_norm = (RMSNorm(self.hd), RMSNorm(self.hd)) if cfg.qk_norm and llama else (None, None)
        self.proj = nn.Linear(d, d, bias=not llama)
        if llama:
            self.gate_up = nn.Linear(d, 2 * cfg.ffn, bias=False)
            self.down = nn.Linear(cfg.ffn, d, bias=False)
        else:
            self.fc = nn.Linear(d, 4 * d)
            self.down = nn.Linear(4 * d, d)

    def _attend(self, x, pos, cu, mask):
        B, T, d = x.shape
        H, kv, hd = self.cfg.n_head, self.kv, self.hd
        llama = self.cfg.style == "llama"
        qkv = self.qkv(self.ln1(x))
        if self.cfg.native:
            q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.view(B * T, d + 2 * kv * hd).split([d, kv * hd, kv * hd], dim=1))
            if llama:
                norms = (None, None) if self.q_norm is None else (self.q_norm.weight, self.k_norm.weight)
                q, k = decoder.head_norm_rope(q, k, *norms, pos, eps=self.q_norm.eps if self.q_norm is not None else 1e-5)
            return decoder.causal_attention(q, k, v, cu).view(B, T, d)
        if kv == H:
            q, k, v = qkv.view(B, T, 3, H, hd).permute(2, 0, 3, 1, 4)
        else:
            q, k, v = (t.view(B, T, -1, hd).transpose(1, 2) for t in qkv.split([d, kv * hd, kv * hd], dim=2))
        if self.q_norm is not None:
            q, k = self.q_norm(q), self.k_norm(k)
        if llama:
            q, k = _rope(q, k, pos=None if pos is None else pos.view(B, T))
        if mask is not None:             # packed sequences: the batch is one row of tokens
            q, k, v = (t.transpose(0, 1).reshape(1, -1, B * T, hd) for t in (q, k, v))
        a = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, is_causal=mask is None, enable_gqa=kv != H)
        if mask is not None:
            a = a.view(H, B, T, hd).transpose(0, 1)
        return a.transpose(1, 2).reshape(B, T, d)

    def forward(self, x, pos=None, cu=None, mask=None):
        x = x + self.proj(self._attend(x, pos, cu, mask))
        h = self.ln2(x)
        if self.cfg.style == "llama":
            g, u = self.gate_up(h).chunk(2, dim=-1)
            x = x + self.down(F.silu(g) * u)
        else:
            x = x + self.down(F.gelu(self.fc(h), approximate="tanh"))
        return x


class GPT(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab, cfg.d_model)
        self.wpe = nn.Embedding(cfg.seq_len, cfg.d_model) if cfg.style == "gpt2" else None
        self.blocks = nn.ModuleList(Block(cfg) for _ in range(cfg.n_layer))
        self.ln_f = RMSNorm(cfg.d_model) if cfg.style == "llama" else nn.LayerNorm(cfg.d_model)
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)
            if getattr(m, "bias", None) is not None:
                nn.init.zeros_(m.bias)

    def forward(self, idx, targets=None, cu_seqlens=None):
        """``idx``, ``targets`` [B, T].  ``cu_seqlens`` (int32 [S + 1], from 0 to B * T): documents packed into the B * T
        tokens, each with positions from 0 (learned positions: the last one stands for all beyond) and attention of its own;
        None: every row of the batch is one."""
        B, T = idx.shape
        native, cu, pos, mask = self.cfg.native, cu_seqlens, None, None
        rows = torch.arange(B * T, device=idx.device) if native or cu is not None else None
        if cu is not None:
            seq = (torch.searchsorted(cu, rows, right=True) - 1).clamp(min=0)
            pos = rows - cu[seq]
            if not native:
                mask = (seq[:, None] == seq[None]) & (rows[:, None] >= rows[None])
        elif native:
            pos = rows % T
            cu = torch.arange(B + 1, device=idx.device, dtype=torch.int32) * T
        x = self.wte(idx)
        if self.wpe is not None:
            x = x + (self.wpe(torch.arange(T, device=idx.device)) if cu_seqlens is None else self.wpe(pos.clamp(0, self.cfg.seq_len - 1)).view(B, T, self.cfg.d_model))
        for blk in self.blocks:
            x = blk(x, pos, cu, mask)
        x = self.ln_f(x)
        if targets is not None and native:
            return decoder.linear_cross_entropy(x, self.wte.weight, targets)
        logits = F.linear(x, self.wte.weight)    # tied output embedding
        if targets is None:
            return logits
        return F.cross_entropy(logits.float().view(-1, logits.size(-1)), targets.view(-1))

    def num_params(self):
        return sum(p.numel() for p in self.parameters())
