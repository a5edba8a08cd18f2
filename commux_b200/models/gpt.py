"""Decoder-only transformer for the DDP workload (12 layers, d_model 768,
12 heads, FFN 3072, vocab 32000, seq 1024): random-init, trained in bf16
autocast with fp32 master weights under torch DDP on the commux backend.

Plain library kernels (cuBLAS GEMMs, flash SDPA) do the math; the backend's
job here is the gradient all-reduce of DDP's buckets, overlapped with the
backward pass on the collective stream.

With ``GPTConfig(act8=True)`` the same weights run through ``commux_b200.ops``
(CUDA only): the residual sums inside the norms, every linear layer's input
but the attention's (which flash SDPA keeps anyway) held in 8 bits for its
weight's gradient, the norms' and GELU's backward passes from those same
checkpoints, and the loss with its gradient in one pass over the logits. Blocks
and layers are the same modules with the same parameters, called as modules, so
hooks and wrappers on them run. Without a gradient nothing is held in 8 bits.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops


@dataclass
class GPTConfig:
    n_layer: int = 12
    n_head: int = 12
    d_model: int = 768
    d_ff: int = 3072
    vocab: int = 32000
    seq_len: int = 1024
    act8: bool = False  # training operators with 8-bit activation checkpoints


class Norm8(nn.LayerNorm):
    def forward(self, x, r=None):
        """(s, y, y's checkpoint) of ``s = x + r`` (s is x when r is None)."""
        pack = torch.is_grad_enabled()
        got = ops.layer_norm(x, self.weight, self.bias, self.eps, residual=r, pack=pack)
        got = got if isinstance(got, tuple) else (got,)
        return x if r is None else got[1], got[0], got[-1] if pack else None


class Linear8(nn.Linear):
    def forward(self, x, act8=None):
        return ops.linear8(x, self.weight, self.bias, act8=act8)


class Block(nn.Module):
    def __init__(self, c: GPTConfig):
        super().__init__()
        norm, linear = (Norm8, Linear8) if c.act8 else (nn.LayerNorm, nn.Linear)
        self.ln1 = norm(c.d_model)
        self.qkv = linear(c.d_model, 3 * c.d_model)
        self.proj = nn.Linear(c.d_model, c.d_model)
        self.ln2 = norm(c.d_model)
        self.fc = linear(c.d_model, c.d_ff)
        self.out = linear(c.d_ff, c.d_model)
        self.n_head = c.n_head
        self.act8 = c.act8

    def forward(self, x, r=None):
        """With ``act8``, the block on the stream ``x`` and what is still to be added
        to it (None before the first block); returns the same pair."""
        if self.act8:
            return self._forward8(x, r)
        x = x + self.proj(self._attend(self.qkv(self.ln1(x))))
        return x + self.out(F.gelu(self.fc(self.ln2(x)), approximate="tanh"))

    def _forward8(self, x, r):
        x, y, kept = self.ln1(x, r)
        r = self.proj(self._attend(self.qkv(y, kept)))
        x, y, kept = self.ln2(x, r)
        h = self.fc(y, kept)
        a, kept = ops.gelu8(h, pack=True) if torch.is_grad_enabled() else (ops.gelu8(h), None)
        return x, self.out(a, kept)

    def _attend(self, qkv):
        B, T, C = qkv.shape[0], qkv.shape[1], qkv.shape[2] // 3
        q, k, v = qkv.split(C, dim=2)
        h = self.n_head
        q = q.view(B, T, h, C // h).transpose(1, 2)
        k = k.view(B, T, h, C // h).transpose(1, 2)
        v = v.view(B, T, h, C // h).transpose(1, 2)
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return y.transpose(1, 2).reshape(B, T, C)


class GPT(nn.Module):
    def __init__(self, c: GPTConfig):
        super().__init__()
        self.c = c
        self.tok = nn.Embedding(c.vocab, c.d_model)
        self.pos = nn.Embedding(c.seq_len, c.d_model)
        self.blocks = nn.ModuleList(Block(c) for _ in range(c.n_layer))
        self.ln = (Norm8 if c.act8 else nn.LayerNorm)(c.d_model)
        self.head = (Linear8 if c.act8 else nn.Linear)(c.d_model, c.vocab, bias=False)
        self.head.weight = self.tok.weight  # tied
        self.apply(self._init)
        for n, p in self.named_parameters():
            if n.endswith("proj.weight") or n.endswith("out.weight"):
                nn.init.normal_(p, 0.0, 0.02 / math.sqrt(2 * c.n_layer))

    @staticmethod
    def _init(m):
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, 0.0, 0.02)
            if m.bias is not None:
                nn.init.zeros_(m.bias)
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, 0.0, 0.02)

    def forward(self, idx, targets=None):
        B, T = idx.shape
        x = self.tok(idx) + self.pos(torch.arange(T, device=idx.device))
        if self.c.act8:
            return self._forward8(x, targets)
        for b in self.blocks:
            x = b(x)
        logits = self.head(self.ln(x))
        if targets is None:
            return logits
        return F.cross_entropy(logits.float().view(-1, logits.size(-1)), targets.view(-1))

    def _forward8(self, x, targets):
        r = None
        for b in self.blocks:
            x, r = b(x, r)
        _, y, kept = self.ln(x, r)
        logits = self.head(y, kept)
        if targets is None:
            return logits
        return ops.cross_entropy(logits, targets)
