"""Fused row-wise LayerNorm on CDNA4 HIP kernels (ops/csrc/ln_kernels.hip).

Drop-in for nn.LayerNorm over the last dimension.  Fast path: CUDA + bf16 +
1-D normalized_shape with D % 256 == 0, D <= 4096 (one wave per row, row in
registers).  Anything else falls back to F.layer_norm, so the same model
runs on CPU for the gloo tests.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import HAVE_EXT, _EXT, _require_ext


class _FusedLN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        shape = x.shape
        D = shape[-1]
        rows = x.numel() // D
        xc = x.contiguous()
        y = torch.empty_like(xc)
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        _EXT.ln_fwd(xc, y, weight, bias, mean, rstd, rows, D, eps)
        ctx.save_for_backward(xc, weight, mean, rstd)
        ctx.dims = (rows, D)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        rows, D = ctx.dims
        dyc = dy.contiguous()
        dx = torch.empty_like(x)
        _EXT.ln_bwd_dx(x, dyc, dx, weight, mean, rstd, rows, D)
        dg32 = torch.empty(D, dtype=torch.float32, device=x.device)
        db32 = torch.empty(D, dtype=torch.float32, device=x.device)
        _EXT.ln_bwd_dgb(x, dyc, mean, rstd, dg32, db32, rows, D)
        return dx, dg32.to(weight.dtype), db32.to(weight.dtype), None


class FusedLayerNorm(nn.LayerNorm):
    def _fast_ok(self, x):
        return (HAVE_EXT and x.is_cuda and x.dtype == torch.bfloat16
                and len(self.normalized_shape) == 1
                and self.normalized_shape[0] % 256 == 0
                and self.normalized_shape[0] <= 4096
                and self.elementwise_affine
                and self.weight is not None and self.bias is not None
                and self.weight.dtype == torch.bfloat16)

    def forward(self, x):
        if self._fast_ok(x):
            return _FusedLN.apply(x, self.weight, self.bias, self.eps)
        return F.layer_norm(x, self.normalized_shape, self.weight, self.bias,
                            self.eps)


# ---------------------------------------------------------------------------
# norms before and after a block with its gate and residual scale
# ---------------------------------------------------------------------------

MAX_JOIN_DIM = 8192


def _norm_plain(f, w, b, kind, eps):
    if kind == "layer":
        f = f - f.mean(-1, keepdim=True)
    f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + eps) * w.to(f.dtype)
    return f if b is None else f + b.to(f.dtype)


def _join_plain(x, u, w, b, gate, pw, pb, scale, eps, kind):
    t = torch.float64 if x.dtype == torch.float64 else torch.float32
    n = u.to(t)
    if pw is not None:
        n = _norm_plain(n, pw, pb, kind, eps)
    if gate is not None:
        n = n * gate.to(t)
    y = x.to(t) * scale + n
    return y.to(x.dtype), _norm_plain(y, w, b, kind, eps).to(x.dtype)


def fused_gated_residual(x, u, weight, bias=None, *, gate=None,
                         post_weight=None, post_bias=None, scale=1.0,
                         eps=1e-5, kind="layer"):
    """A sublayer's end and the next one's beginning in one pass:

        n = Post(u) if post_weight is given, else u
        y = scale * x + gate * n          (the residual stream)
        h = Norm(y)                       (input of the next sublayer)

    Returns (y, h).  x, u: [..., D] of one type; ``weight``/``bias`` and
    ``post_weight``/``post_bias``: [D] of that type; ``kind``: "layer" or "rms"
    for both norms.  ``gate``: None, [D], [B, 1, D] for x of [B, T, D], or x's
    shape.  The norm is taken of y before its rounding.

    GPU: HIP kernels (ops/csrc/join_kernels.hip) for bf16 and fp32, D up to
    8192, gates of fewer than 2**23 samples; other types or sizes raise.  CPU:
    plain torch, the oracle.
    """
    if kind not in ("layer", "rms"):
        raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
    if x.dim() < 1 or x.shape != u.shape:
        raise ValueError(f"x {tuple(x.shape)} and u {tuple(u.shape)} must "
                         "have one shape")
    D = x.shape[-1]
    if D < 1:
        raise ValueError("rows must have at least one element")
    if post_bias is not None and post_weight is None:
        raise ValueError("post_bias needs post_weight")
    for name, t in (("weight", weight), ("bias", bias),
                    ("post_weight", post_weight), ("post_bias", post_bias)):
        if t is not None and tuple(t.shape) != (D,):
            raise ValueError(f"{name} must be [{D}], got {tuple(t.shape)}")
    for name, t in (("u", u), ("weight", weight), ("bias", bias),
                    ("post_weight", post_weight), ("post_bias", post_bias),
                    ("gate", gate)):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{name} must have x's type and device")
    groups, gate_kind = 1, 0
    if gate is not None:
        if tuple(gate.shape) == (D,):
            gate_kind = 1
        elif gate.shape == x.shape:
            gate_kind = 2
        elif x.dim() == 3 and tuple(gate.shape) == (x.shape[0], 1, D):
            gate_kind, groups = 1, x.shape[0]
        else:
            raise ValueError(
                f"gate must be [{D}], [B, 1, {D}] or x's shape, got "
                f"{tuple(gate.shape)}")
    if _require_ext(x) and x.numel():
        if x.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("fused_gated_residual on GPU: bf16 or fp32")
        if D > MAX_JOIN_DIM:
            raise ValueError(f"fused_gated_residual on GPU: rows of at most "
                             f"{MAX_JOIN_DIM}, got {D}")
        return tuple(_EXT.gated_residual(
            x, u, weight, bias, gate, post_weight, post_bias, float(scale),
            float(eps), kind == "layer", groups, gate_kind))
    return _join_plain(x, u, weight, bias, gate, post_weight, post_bias,
                       scale, eps, kind)
