"""What the transformer blocks share: two branches, attention and mlp, each
added to the residual stream, with or without gates."""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.ln import fused_gated_residual


class TwoBranches(nn.Module):
    """A subclass brings ``attend``, n1, n2, fc1 and fc2.

    Gates (layer_scale): one for each channel of both branches.  The norms then
    ride with gate and residual in one pass (``joined``): a model calls its
    blocks, but of its norm modules only the first; the others lend their
    weights, and hooks on them do not run.
    """

    def add_gates(self, dim, layer_scale):
        self.g1 = self.g2 = None
        if layer_scale is not None:
            self.g1 = nn.Parameter(torch.full((dim,), float(layer_scale)))
            self.g2 = nn.Parameter(torch.full((dim,), float(layer_scale)))

    def mlp(self, h):
        return self.fc2(F.gelu(self.fc1(h)))

    def forward(self, x, pos=None, h=None, after=None):
        """x -> x behind this block; with h and ``after``: see ``joined``."""
        if after is not None:
            return self.joined(x, h, after, pos)
        u = self.attend(self.n1(x), pos)
        if self.g1 is None:
            x = x + u
            return x + self.mlp(self.n2(x))
        x, h = self._join(x, u, self.g1, self.n2)
        return x + self.g2 * self.mlp(h)

    def joined(self, x, h, after, pos=None):
        """x: residual stream, h: its norm n1.  Returns the stream behind this
        block and its norm by ``after``."""
        x, h = self._join(x, self.attend(h, pos), self.g1, self.n2)
        return self._join(x, self.mlp(h), self.g2, after)

    @staticmethod
    def _join(x, u, gate, norm):
        # under autocast a branch comes back in fewer bits than the stream has
        return fused_gated_residual(x, u.to(x.dtype), norm.weight, norm.bias,
                                    gate=gate, eps=norm.eps)
