"""Llama-style decoder for the Muon benchmark: RMSNorm, rotary position embedding, causal attention (key / value heads may be fewer than
query heads), SwiGLU MLP, untied output head.  ``Llama(ids)`` takes rows of one length; with ``cu_seqlens`` the ids are one row of documents
of different lengths, each with positions and attention of its own.  ``Llama.loss`` is the training loss without stored logits.  The 1.3 B configuration is 24 layers, d_model 2048, 16 heads, MLP 5504,
vocabulary 32000 (1,345,423,360 parameters, 168 two-dimensional block weights)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import nn_ops


@dataclass
class LlamaConfig:
    n_layers: int = 24
    d_model: int = 2048
    n_heads: int = 16
    d_ff: int = 5504
    vocab: int = 32000
    max_seq: int = 2048
    rope_theta: float = 10000.0
    eps: float = 1e-5
    n_kv_heads: Optional[int] = None                                    # None: as many as n_heads


LLAMA_1P3B = LlamaConfig()
LLAMA_TINY = LlamaConfig(n_layers=2, d_model=128, n_heads=4, d_ff=352, vocab=256, max_seq=64)


class RMSNorm(nn.Module):
    def __init__(self, d, eps=1e-5):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d))
        self.eps = eps

    def forward(self, x):
        return nn_ops.rms_norm(x, None, self.weight, self.eps)

    def add_norm(self, x, residual):
        """(RMSNorm(x + residual), x + residual); on CUDA one kernel does the add, the statistics and the scaling."""
        if residual is None:
            return self.forward(x), x
        return nn_ops.norm_residual(x, residual, self.weight, None, self.eps, rms=True)


def rope_tables(seq, hd, theta, device, dtype=torch.float32):
    inv = 1.0 / (theta ** (torch.arange(0, hd, 2, device=device, dtype=torch.float32) / hd))
    ang = torch.outer(torch.arange(seq, device=device, dtype=torch.float32), inv)
    return ang.cos().to(dtype), ang.sin().to(dtype)


class LlamaBlock(nn.Module):
    def __init__(self, cfg: LlamaConfig):
        super().__init__()
        d = cfg.d_model
        self.h, self.kv = cfg.n_heads, cfg.n_kv_heads or cfg.n_heads
        if self.h % self.kv:
            raise ValueError(f"{self.h} query heads are not a multiple of {self.kv} key heads")
        d_kv = d // self.h * self.kv
        self.attn_norm, self.mlp_norm = RMSNorm(d, cfg.eps), RMSNorm(d, cfg.eps)
        self.wq, self.wk, self.wv, self.wo = (nn.Linear(d, n, bias=False) for n in (d, d_kv, d_kv, d))
        self.w_gate, self.w_up = nn.Linear(d, cfg.d_ff, bias=False), nn.Linear(d, cfg.d_ff, bias=False)
        self.w_down = nn.Linear(cfg.d_ff, d, bias=False)

    def forward(self, x, pending, cos, sin, cu_seqlens=None):
        """The residual stream entering the block is x + pending (pending = the previous block's MLP output, not yet added:
        the add is fused into this block's first norm).  Returns the same pair for the next block."""
        B, S, D = x.shape
        y, x = self.attn_norm.add_norm(x, pending)
        q, k, v = (w(y).view(B, S, h, D // self.h) for w, h in ((self.wq, self.h), (self.wk, self.kv), (self.wv, self.kv)))
        q, k = nn_ops.rope(q, cos, sin), nn_ops.rope(k, cos, sin)
        if cu_seqlens is None:
            o = nn_ops.attention(q, k, v, causal=True)                  # [B, S, H, hd]
        else:
            o = nn_ops.attention_packed(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), cu_seqlens)
        y, x = self.mlp_norm.add_norm(self.wo(o.reshape(B, S, D)), x)
        return x, self.w_down(nn_ops.swiglu(self.w_gate(y), self.w_up(y)))


class Llama(nn.Module):
    def __init__(self, cfg: LlamaConfig = LLAMA_1P3B):
        super().__init__()
        self.cfg = cfg
        self.embed = nn.Embedding(cfg.vocab, cfg.d_model)
        self.layers = nn.ModuleList([LlamaBlock(cfg) for _ in range(cfg.n_layers)])
        self.norm = RMSNorm(cfg.d_model, cfg.eps)
        self.lm_head = nn.Linear(cfg.d_model, cfg.vocab, bias=False)

    def hidden(self, ids, cu_seqlens: Optional[torch.Tensor] = None):
        """What the head reads: [..., d_model] for ids [B, S], or for packed ids [T] or [1, T] with the offsets ``cu_seqlens`` of their
        documents (int32 or int64, on the ids' device).  Rows of no document attend to nothing."""
        cfg = self.cfg
        shape = ids.shape
        if cu_seqlens is not None:
            if ids.numel() != ids.shape[-1]:
                raise ValueError(f"packed ids are one row of tokens, got {tuple(shape)}")
            ids = ids.reshape(1, -1)
        B, S = ids.shape
        cos, sin = rope_tables(S, cfg.d_model // cfg.n_heads, cfg.rope_theta, ids.device)
        if cu_seqlens is not None:
            cu_seqlens = cu_seqlens.to(torch.int32)
            pos = nn_ops.packed_positions(cu_seqlens, S)
            cos, sin = cos[pos], sin[pos]
        elif (cfg.n_kv_heads or cfg.n_heads) != cfg.n_heads:            # rows of one length are documents too
            cu_seqlens = torch.arange(0, (B + 1) * S, S, dtype=torch.int32, device=ids.device) if S else torch.zeros(1, dtype=torch.int32, device=ids.device)
        h = nn_ops.embedding(ids, self.embed.weight)
        pending = None
        for l in self.layers:
            h, pending = l(h, pending, cos, sin, cu_seqlens)
        return self.norm.add_norm(h, pending)[0].reshape(*shape, cfg.d_model)

    def forward(self, ids, cu_seqlens: Optional[torch.Tensor] = None):
        return self.lm_head(self.hidden(ids, cu_seqlens))

    def loss(self, ids, targets, cu_seqlens: Optional[torch.Tensor] = None, ignore_index: int = -100):
        """Mean cross-entropy of ``forward(ids, cu_seqlens)`` against ``targets`` (shaped like ids) without storing the logits."""
        return nn_ops.linear_cross_entropy(self.hidden(ids, cu_seqlens), self.lm_head.weight, targets, ignore_index)

    def matrix_params(self):
        """2-D weights of the blocks (Muon group); everything else (embedding, head, norms) goes to AdamW."""
        return [p for l in self.layers for p in l.parameters() if p.dim() == 2]

    def other_params(self):
        ids = {id(p) for p in self.matrix_params()}
        return [p for p in self.parameters() if id(p) not in ids]
