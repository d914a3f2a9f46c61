"""Fused flash attention (MFMA-tiled, ops/csrc/mfma_attn_kernels.hip).

Two in-tree implementations, selected by PS_AMD_ATTN:
  "mfma" (default) — 16x16x32-MFMA-tiled flash fwd+bwd, 128-row blocks,
                     transposed-operand LDS staging (round 2);
  "ref"            — the one-wave-per-row correctness kernels
                     (attn_kernels.hip) — the on-GPU oracle;
  "torch"          — torch SDPA (aotriton).

Shape contract for the fused paths: [B, H, N, D] bf16 contiguous, D == 64
(GPT-2-small and ViT-B/16 head dim).  Anything else falls back to torch
SDPA.

``fused_window_sdpa`` is causal attention with a sliding window and first
tokens that stay visible (ops/csrc/window_attn_kernels.hip): grouped heads,
D 64 or 128, padded batches.
"""

from __future__ import annotations

import math
import os

import torch
import torch.nn.functional as F

from . import HAVE_EXT, _EXT, _require_ext


def _impl():
    return os.environ.get("PS_AMD_ATTN", "mfma")


class _FusedSDPA(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, use_mfma):
        B, H, N, D = q.shape
        scale = 1.0 / math.sqrt(D)
        # explicit shape: empty_like would inherit q's (possibly strided)
        # layout, and o is always written contiguous
        o = torch.empty((B, H, N, D), dtype=q.dtype, device=q.device)
        lse = torch.empty(B * H * N, dtype=torch.float32, device=q.device)
        if use_mfma:
            _EXT.fa_fwd(q, k, v, o, lse, N, scale, causal)
        else:
            _EXT.attn_fwd(q, k, v, o, lse, N, scale, causal)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.causal = causal
        ctx.use_mfma = use_mfma
        return o

    @staticmethod
    def backward(ctx, dout):
        q, k, v, o, lse = ctx.saved_tensors
        B, H, N, D = q.shape
        scale = 1.0 / math.sqrt(D)
        dout = dout.contiguous()
        delta = torch.empty_like(lse)
        dq = torch.empty((B, H, N, D), dtype=q.dtype, device=q.device)
        dk = torch.empty_like(dq)
        dv = torch.empty_like(dq)
        if ctx.use_mfma:
            _EXT.fa_bwd(q, k, v, o, dout, lse, delta, dq, dk, dv, N, scale,
                        ctx.causal)
        else:
            _EXT.attn_bwd(q, k, v, o, dout, lse, delta, dq, dk, dv, N, scale,
                          ctx.causal)
        return dq, dk, dv, None, None


class _FusedSDPAQkv(torch.autograd.Function):
    """Attention on a FUSED [B,T,3,H,D] qkv tensor: forward slices q/k/v as
    strided views (no copies); backward writes dq/dk/dv STRIDED into one
    dqkv buffer, so the gradient of the qkv projection arrives assembled —
    autograd's CatArrayBatchedCopy pass (~2 ms/step on GPT-2-small,
    profiles/gpt2_steady_r02.md) disappears."""

    @staticmethod
    def forward(ctx, qkv, causal):
        B, T, three, H, D = qkv.shape
        q, k, v = (qkv[:, :, i].permute(0, 2, 1, 3) for i in range(3))
        scale = 1.0 / math.sqrt(D)
        o = torch.empty((B, H, T, D), dtype=qkv.dtype, device=qkv.device)
        lse = torch.empty(B * H * T, dtype=torch.float32, device=qkv.device)
        _EXT.fa_fwd(q, k, v, o, lse, T, scale, causal)
        ctx.save_for_backward(qkv, o, lse)
        ctx.causal = causal
        return o

    @staticmethod
    def backward(ctx, dout):
        qkv, o, lse = ctx.saved_tensors
        B, T, three, H, D = qkv.shape
        q, k, v = (qkv[:, :, i].permute(0, 2, 1, 3) for i in range(3))
        scale = 1.0 / math.sqrt(D)
        dout = dout.contiguous()
        delta = torch.empty_like(lse)
        dqkv = torch.empty_like(qkv)
        dq, dk, dv = (dqkv[:, :, i].permute(0, 2, 1, 3) for i in range(3))
        _EXT.fa_bwd(q, k, v, o, dout, lse, delta, dq, dk, dv, T, scale,
                    ctx.causal)
        return dqkv, None


def fused_sdpa_qkv(qkv, is_causal=False):
    """Attention for a fused qkv projection output [B, T, 3, H, D] (D==64).
    Returns [B, H, T, D].  Falls back to slicing + fused_sdpa."""
    if (_impl() == "mfma" and HAVE_EXT and qkv.is_cuda
            and qkv.dtype == torch.bfloat16 and qkv.dim() == 5
            and qkv.shape[2] == 3 and qkv.shape[-1] == 64
            and qkv.is_contiguous()):
        return _FusedSDPAQkv.apply(qkv, bool(is_causal))
    q, k, v = qkv.permute(2, 0, 3, 1, 4)
    return fused_sdpa(q, k, v, is_causal=is_causal)


def fused_sdpa(q, k, v, is_causal=False):
    """Like F.scaled_dot_product_attention for [B,H,N,D] with D==64."""
    impl = _impl()
    if (impl in ("mfma", "ref") and HAVE_EXT and q.is_cuda
            and q.dtype == torch.bfloat16
            and q.dim() == 4 and q.shape[-1] == 64
            and q.shape == k.shape == v.shape):
        mfma = impl == "mfma"
        if mfma and (q.stride(-1) == 1 and q.stride(0) % 8 == 0
                     and q.stride(1) % 8 == 0 and q.stride(2) % 8 == 0
                     and q.stride() == k.stride() == v.stride()):
            # the MFMA kernels read strided q/k/v natively (e.g. head
            # slices of a fused qkv projection) — no copies
            return _FusedSDPA.apply(q, k, v, bool(is_causal), True)
        return _FusedSDPA.apply(q.contiguous(), k.contiguous(),
                                v.contiguous(), bool(is_causal), mfma)
    return F.scaled_dot_product_attention(q, k, v, is_causal=is_causal)


# ---------------------------------------------------------------------------
# sliding window with first tokens that stay visible
# ---------------------------------------------------------------------------

class _Product(torch.autograd.Function):
    """a @ b in their own type: autocast would make both passes bf16."""

    generate_vmap_rule = True

    @staticmethod
    def forward(a, b):
        with torch.autocast(a.device.type, enabled=False):
            return a @ b

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(*inputs)

    @staticmethod
    def backward(ctx, g):
        a, b = ctx.saved_tensors
        with torch.autocast(a.device.type, enabled=False):
            return g @ b.transpose(-2, -1), a.transpose(-2, -1) @ g


def _window_plain(q, k, v, window, sinks, lengths, scale):
    """The whole score matrix in fp32 (fp64 for fp64): oracle, and the path of
    types and head sizes that have no kernel."""
    B, H, N, D = q.shape
    G = H // k.shape[1]
    t = torch.float64 if q.dtype == torch.float64 else torch.float32
    kf = k.to(t).repeat_interleave(G, 1)
    vf = v.to(t).repeat_interleave(G, 1)
    i = torch.arange(N, device=q.device)[:, None]
    j = torch.arange(N, device=q.device)[None]
    vis = ((j <= i) & ((i - j < window) | (j < sinks)))[None]
    if lengths is not None:
        n = lengths.long().clamp(0, N)[:, None, None]
        vis = vis & (i < n) & (j < n)
        # what stands behind a sequence is not looked at, NaN included
        past = (torch.arange(N, device=q.device) >= n[:, 0])[:, None, :, None]
        q, kf, vf = (x.masked_fill(past, 0) for x in (q, kf, vf))
    z = _Product.apply(q.to(t), kf.transpose(2, 3).contiguous()) * scale
    z = z.masked_fill(~vis[:, None], -math.inf)
    # a row of no keys has no maximum
    top = z.detach().amax(3, keepdim=True) if N else z.detach().sum(3, True)
    e = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top),
                                  top))
    total = e.sum(3, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    o = _Product.apply(p, vf)
    if lengths is not None:
        # nor is a gradient that comes from there
        o = o.masked_fill(past, 0)
    return o.to(q.dtype).transpose(1, 2).contiguous().transpose(1, 2)


def fused_window_sdpa(q, k, v, window, sinks=0, lengths=None, scale=None):
    """Causal attention in which row i sees key j <= i if ``i - j < window`` or
    ``j < sinks`` (the first tokens stay visible).

    q: [B, H, N, D]; k, v: [B, KV, N, D] with H a multiple of KV (each key head
    serves H/KV neighbouring query heads).  ``lengths``: optional int32 [B] on
    the same device; rows and keys from a sequence's length on do not exist:
    they may hold anything, their outputs and gradients are zero.  ``scale``:
    positive, 1/sqrt(D) by default.  Returns [B, H, N, D], stored with the
    heads behind the rows.

    GPU, bf16, D 64 or 128: MFMA kernels forward and backward
    (ops/csrc/window_attn_kernels.hip), reading any strides with unit d stride
    and 16-byte rows.  Anything else: plain torch with the whole score matrix.
    Where a gradient will be asked for, a second tensor of the output's size is
    kept for it.
    Values inside the lengths must be finite: a product with a weight of zero
    lets a NaN or infinity reach rows that do not see it.
    """
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q must be [B, H, N, D], k and v [B, KV, N, D]")
    B, H, N, D = q.shape
    if k.shape[0] != B or k.shape[2] != N or k.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ "
                         "in B, N or D")
    if D < 1:
        raise ValueError("heads must have at least one element")
    if k.shape[1] < 1 or H % k.shape[1]:
        raise ValueError(f"{H} query heads do not divide over {k.shape[1]} "
                         "key heads")
    if not (q.dtype == k.dtype == v.dtype and q.is_floating_point()):
        raise ValueError("q, k and v must have one floating type")
    if not (q.device == k.device == v.device):
        raise ValueError("q, k and v must be on one device")
    window, sinks = int(window), int(sinks)
    if window < 1 or sinks < 0:
        raise ValueError("window must be 1 or more, sinks 0 or more")
    if lengths is not None and (lengths.dtype != torch.int32
                                or tuple(lengths.shape) != (B,)
                                or lengths.device != q.device):
        raise ValueError(f"lengths must be int32 [{B}] on q's device")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    if (_require_ext(q) and q.dtype == torch.bfloat16 and D in (64, 128)
            and q.numel()):
        return _EXT.window_sdpa(q, k, v, window, sinks, lengths, scale)
    return _window_plain(q, k, v, window, sinks, lengths, scale)
