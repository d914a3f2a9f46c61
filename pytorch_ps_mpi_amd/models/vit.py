"""ViT-B/16 (Dosovitskiy et al. 2020) for BASELINE config 4."""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.attn import fused_sdpa, fused_sdpa_qkv
from ..ops.linear import FusedLinear
from ..ops.ln import FusedLayerNorm
from ..ops.rope import AxialRotary
from .block import TwoBranches


class Block(TwoBranches):
    """rotary : AxialRotary that turns q and k by height and width;
    layer_scale : start value of the gates (models/block.py)."""

    def __init__(self, dim, heads, mlp_ratio=4.0, rotary=None,
                 layer_scale=None):
        super().__init__()
        self.n1 = FusedLayerNorm(dim)
        self.qkv = FusedLinear(dim, dim * 3)
        self.proj = FusedLinear(dim, dim)
        self.heads = heads
        self.rotary = rotary
        self.n2 = FusedLayerNorm(dim)
        h = int(dim * mlp_ratio)
        self.fc1 = FusedLinear(dim, h)
        self.fc2 = FusedLinear(h, dim)
        self.add_gates(dim, layer_scale)

    def attend(self, h, pos=None):
        B, N, D = h.shape
        qkv = self.qkv(h).view(B, N, 3, self.heads, D // self.heads)
        if self.rotary is None:
            y = fused_sdpa_qkv(qkv)  # [B, H, N, Dh]
        else:
            q, k, v = qkv.unbind(2)
            q, k = self.rotary(q, k, pos)
            y = fused_sdpa(q.transpose(1, 2), k.transpose(1, 2),
                           v.transpose(1, 2))
        return self.proj(y.transpose(1, 2).reshape(B, N, D))


class ViT(nn.Module):
    """rotary=True: patches carry their row and column by rotary positions
    (beside the learned ones); layer_scale: see Block."""

    def __init__(self, img=224, patch=16, dim=768, depth=12, heads=12,
                 num_classes=1000, rotary=False, layer_scale=None):
        super().__init__()
        # patch embedding as unfold + Linear: with stride == kernel the
        # "conv" is a pure reshape + GEMM, which keeps it on hipBLASLt
        # (MIOpen's stride-16 bf16 conv fell back to naive/im2col kernels —
        # 60% of the step in the round-1 profile)
        self.patch = patch
        self.patch_embed = nn.Linear(3 * patch * patch, dim)
        n = (img // patch) ** 2
        self.cls = nn.Parameter(torch.zeros(1, 1, dim))
        self.pos = nn.Parameter(torch.randn(1, n + 1, dim) * 0.02)
        rot = None
        if rotary:
            pairs = dim // heads // 4
            rot = AxialRotary(dim // heads, (pairs, pairs))
            side = torch.arange(img // patch)
            grid = torch.stack([side.repeat_interleave(len(side)),
                                side.repeat(len(side))]) + 1
            # the class token stands at (0, 0)
            self.register_buffer("grid", F.pad(grid, (1, 0)),
                                 persistent=False)
        self.rotary = rotary
        self.layer_scale = layer_scale
        self.blocks = nn.ModuleList(
            Block(dim, heads, rotary=rot, layer_scale=layer_scale)
            for _ in range(depth))
        self.norm = FusedLayerNorm(dim)
        self.head = nn.Linear(dim, num_classes)

    def _patchify(self, x):
        B, C, H, W = x.shape
        p = self.patch
        x = x.view(B, C, H // p, p, W // p, p)
        x = x.permute(0, 2, 4, 1, 3, 5).reshape(B, (H // p) * (W // p),
                                                C * p * p)
        return x

    def forward(self, x):
        x = self.patch_embed(self._patchify(x))
        cls = self.cls.expand(x.shape[0], -1, -1)
        x = torch.cat([cls, x], dim=1) + self.pos
        pos = self.grid if self.rotary else None
        if self.layer_scale is None:
            for blk in self.blocks:
                x = blk(x, pos)
            return self.head(self.norm(x)[:, 0])
        norms = [blk.n1 for blk in self.blocks] + [self.norm]
        h = norms[0](x)
        for blk, after in zip(self.blocks, norms[1:]):
            x, h = blk(x, pos, h, after)
        return self.head(h[:, 0])


def vit_b16(num_classes=1000, **kw):
    return ViT(dim=768, depth=12, heads=12, num_classes=num_classes, **kw)
