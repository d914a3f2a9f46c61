"""GPT-2-small (Radford et al. 2019) for BASELINE config 5
(AsySG-InCon stale-gradient path)."""

from __future__ import annotations


import torch
import torch.nn as nn

from ..ops.attn import fused_sdpa_qkv, fused_window_sdpa
from ..ops.ce import fused_cross_entropy
from ..ops.linear import FusedLinear
from ..ops.ln import FusedLayerNorm
from ..ops.rope import AxialRotary
from .block import TwoBranches


class CausalBlock(TwoBranches):
    """One transformer block.

    window, sinks : attention to the last ``window`` tokens and the first
        ``sinks`` ones; kv_heads : key heads, each shared by heads/kv_heads
        query heads; rotary : AxialRotary that turns q and k.  Any of them
        takes the windowed kernels, none the full causal ones.
    layer_scale : start value of the gates (models/block.py).
    """

    def __init__(self, dim, heads, window=None, sinks=0, kv_heads=None,
                 rotary=None, layer_scale=None):
        super().__init__()
        self.n1 = FusedLayerNorm(dim)
        self.local = not (window is None and kv_heads is None
                          and rotary is None)
        self.window, self.sinks = window, sinks
        self.kv_heads = heads if kv_heads is None else kv_heads
        self.rotary = rotary
        self.qkv = FusedLinear(
            dim, dim // heads * (heads + 2 * self.kv_heads))
        self.proj = FusedLinear(dim, dim)
        self.n2 = FusedLayerNorm(dim)
        self.fc1 = FusedLinear(dim, 4 * dim)
        self.fc2 = FusedLinear(4 * dim, dim)
        self.heads = heads
        self.add_gates(dim, layer_scale)

    def attend(self, h, pos=None):
        B, T, D = h.shape
        hd = D // self.heads
        if not self.local:
            qkv = self.qkv(h).view(B, T, 3, self.heads, hd)
            y = fused_sdpa_qkv(qkv, is_causal=True)  # [B, H, T, Dh]
        else:
            kv = self.kv_heads
            q, k, v = self.qkv(h).view(B, T, -1, hd).split(
                [self.heads, kv, kv], 2)
            if self.rotary is not None:
                if pos is None:
                    pos = torch.arange(T, device=h.device)[None]
                q, k = self.rotary(q, k, pos)
            y = fused_window_sdpa(q.transpose(1, 2), k.transpose(1, 2),
                                  v.transpose(1, 2),
                                  T if self.window is None else self.window,
                                  self.sinks)
        return self.proj(y.transpose(1, 2).reshape(B, T, D))


class GPT2(nn.Module):
    """window, sinks, kv_heads, layer_scale: see CausalBlock; rotary=True
    takes rotary positions in place of learned ones."""

    def __init__(self, vocab=50257, ctx=1024, dim=768, depth=12, heads=12,
                 window=None, sinks=0, kv_heads=None, rotary=False,
                 layer_scale=None):
        super().__init__()
        if dim % heads or (kv_heads is not None and
                           (kv_heads < 1 or heads % kv_heads)):
            raise ValueError("heads must divide dim, kv_heads must divide "
                             "heads")
        if (window is not None and window < 1) or sinks < 0:
            raise ValueError("window must be 1 or more, sinks 0 or more")
        self.wte = nn.Embedding(vocab, dim)
        rot = AxialRotary(dim // heads, (dim // heads // 2,)) if rotary \
            else None
        self.wpe = None if rotary else nn.Embedding(ctx, dim)
        self.blocks = nn.ModuleList(
            CausalBlock(dim, heads, window, sinks, kv_heads, rot, layer_scale)
            for _ in range(depth))
        self.norm = FusedLayerNorm(dim)
        self.ctx = ctx
        self.layer_scale = layer_scale
        for m in self.modules():
            if isinstance(m, nn.Linear):
                nn.init.normal_(m.weight, std=0.02)
                if m.bias is not None:
                    nn.init.zeros_(m.bias)
            elif isinstance(m, nn.Embedding):
                nn.init.normal_(m.weight, std=0.02)

    def forward(self, idx):
        B, T = idx.shape
        pos = torch.arange(T, device=idx.device)
        x = self.wte(idx)
        if self.wpe is not None:
            x = x + self.wpe(pos)[None]
        pos = pos[None]  # one axis
        if self.layer_scale is None:
            for blk in self.blocks:
                x = blk(x, pos)
            x = self.norm(x)
        else:
            norms = [blk.n1 for blk in self.blocks] + [self.norm]
            h = norms[0](x)
            for blk, after in zip(self.blocks, norms[1:]):
                x, h = blk(x, pos, h, after)
            x = h
        # tied output head
        return x @ self.wte.weight.t()

    def loss(self, idx, targets):
        # CE directly on the bf16 logits: torch's log_softmax accumulates in
        # fp32 internally; materializing a fp32 [tokens, vocab] copy cost
        # ~12 ms/step at batch 96 (9.9 GB of extra traffic).
        logits = self.forward(idx)
        return fused_cross_entropy(
            logits.reshape(-1, logits.size(-1)).contiguous(),
            targets.reshape(-1))


def gpt2_small(vocab=50304, ctx=1024, **kw):
    # vocab padded 50257 -> 50304 (multiple of 64) for GEMM tile alignment
    return GPT2(vocab=vocab, ctx=ctx, **kw)
