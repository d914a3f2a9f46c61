"""Rotary positions with several axes (ops/csrc/rope_kernels.hip).

For text one axis, for images height and width, for video time, height and
width: the first 2*P elements of a head are P pairs, ``sections`` says how many
of them turn with each axis, the rest of the head passes through.  Angles are
computed in 64 bits, so far positions keep theirs.  Stands before
``fused_sdpa`` / ``fused_window_sdpa``.

GPU: the HIP kernel for bf16, fp16 and fp32 tensors of any strides with unit
last stride.  CPU: plain torch, the oracle.
"""

from __future__ import annotations

import math

import torch

from . import _EXT, _require_ext

MAX_PAIRS = 256
MAX_AXES = 4
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _rotate_plain(x, cos, sin, interleaved):
    P = cos.shape[-1]
    f = x.float()
    r, rest = f[..., :2 * P], f[..., 2 * P:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = r[..., :P], r[..., P:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, rest], -1).to(x.dtype)


class AxialRotary:
    """Rotary embedding of q and k by positions on several axes.

    head_dim : elements of a head; sections : pairs of each axis (1 to 4 axes,
        ``2 * sum(sections) <= head_dim``, at most 256 pairs).
    base : pair i of an axis with n pairs has frequency ``base**(-i/n)``; with
        ``shared=True`` the pairs of all axes count through:
        ``base**(-p/sum(sections))`` for pair p.
    interleaved : pairs are elements (2p, 2p+1); else (p, P+p).

    ``rot(q, k, positions)`` -> rotated copies of q [B,N,H,D] and k [B,N,KV,D];
    positions: int32/int64 [axes, B, N], or [axes, N] for all of a batch.
    """

    def __init__(self, head_dim, sections, base=10000.0, shared=False,
                 interleaved=False):
        sections = tuple(int(s) for s in sections)
        if not 1 <= len(sections) <= MAX_AXES or min(sections) < 1:
            raise ValueError(f"sections: 1 to {MAX_AXES} axes of one pair or "
                             f"more, got {sections}")
        P = sum(sections)
        if 2 * P > head_dim or P > MAX_PAIRS:
            raise ValueError(f"{P} pairs do not fit a head of {head_dim} "
                             f"(and at most {MAX_PAIRS})")
        if not base > 0:
            raise ValueError("base must be positive")
        self.head_dim, self.sections = int(head_dim), sections
        self.interleaved = bool(interleaved)
        if shared:
            f = [base ** (-p / P) for p in range(P)]
        else:
            f = [base ** (-i / n) for n in sections for i in range(n)]
        self.freq = torch.tensor(f, dtype=torch.float64)  # radians a position
        self._rev = self.freq / (2 * math.pi)
        ends = [sum(sections[:i + 1]) for i in range(3)]
        self._start = [min(e, P) if i + 1 < len(sections) else P
                       for i, e in enumerate(ends)]

    def _check(self, q, k, positions):
        if q.dim() != 4 or k.dim() != 4:
            raise ValueError("q and k must be [B, N, H, D] and [B, N, KV, D]")
        if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} "
                             "differ in B, N or D")
        if q.shape[3] != self.head_dim:
            raise ValueError(f"made for heads of {self.head_dim}, got "
                             f"{q.shape[3]}")
        if q.dtype != k.dtype or q.dtype not in _DTYPE:
            raise ValueError("q and k must both be bf16, fp16 or fp32")
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("positions must be int32 or int64")
        if positions.dim() == 2:
            positions = positions[:, None].expand(-1, q.shape[0], -1)
        if tuple(positions.shape) != (len(self.sections), *q.shape[:2]):
            raise ValueError(
                f"positions must be [{len(self.sections)}, B, N] or "
                f"[{len(self.sections)}, N], got {tuple(positions.shape)}")
        if not (q.device == k.device == positions.device):
            raise ValueError("q, k and positions must be on one device")
        return positions

    def __call__(self, q, k, positions):
        positions = self._check(q, k, positions)
        if _require_ext(q):
            return tuple(_EXT.rope(q, k, positions, self._start, self._rev,
                                   self.interleaved))
        cos, sin = self._angles(positions)
        return (_rotate_plain(q, cos, sin, self.interleaved),
                _rotate_plain(k, cos, sin, self.interleaved))

    def _angles(self, positions):
        axis = torch.repeat_interleave(
            torch.arange(len(self.sections)), torch.tensor(self.sections))
        t = positions.double()[axis].permute(1, 2, 0) * self.freq
        return torch.cos(t).float()[:, :, None], \
            torch.sin(t).float()[:, :, None]
