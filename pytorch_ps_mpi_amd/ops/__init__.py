"""Device-dispatching op layer.

On GPU (ROCm) every function calls the in-tree gfx950 HIP extension
(`_ps_hip.so`) and FAILS LOUDLY if it is missing — there is no silent eager
fallback on a GPU box.  On CPU the same semantics are provided by plain torch
reference implementations (used by the gloo multi-process tests and as the
numerics oracle for the HIP kernels).

These ops replace the reference's Python hot path
(stsievert/pytorch_ps_mpi): cross-rank grad sum ps.py:176, SGD math
ps.py:197-214, Adam math ps.py:218-261, and the external `codings`
compression plugin (ps.py:18).
"""

from __future__ import annotations

import math

import torch

_EXT = None
_EXT_ERR = None
try:
    from . import _ps_hip as _EXT  # type: ignore
except Exception as e:  # pragma: no cover - exercised only without built ext
    _EXT_ERR = e

HAVE_EXT = _EXT is not None

QCHUNK = 256
TOPK_WS_WORDS = 2048 + 4 + 2 * 2048


def _require_ext(t: torch.Tensor):
    if t.is_cuda:
        if not HAVE_EXT:
            raise RuntimeError(
                "pytorch_ps_mpi_amd HIP extension (_ps_hip) is not built but a "
                "GPU tensor reached the op layer. Build it with "
                "`PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace`. "
                f"Import error was: {_EXT_ERR!r}"
            )
        return True
    return False


# ---------------------------------------------------------------------------
# fused optimizers
# ---------------------------------------------------------------------------

def fused_sgd(p, buf, g, p_out, *, lr, momentum=0.0, dampening=0.0, wd=0.0,
              nesterov=False, mom_init=False, gscale=1.0):
    """p/buf/g are flat fp32; p_out optional bf16/f32 model copy."""
    if _require_ext(p):
        _EXT.fused_sgd(p, buf, g, p_out, lr, momentum, dampening, wd,
                       bool(nesterov), bool(mom_init), gscale)
        return
    d = g * gscale
    if wd != 0.0:
        d = d.add(p, alpha=wd)
    if momentum != 0.0:
        if mom_init:
            buf.copy_(d)
        else:
            buf.mul_(momentum).add_(d, alpha=1.0 - dampening)
        d = d.add(buf, alpha=momentum) if nesterov else buf
    p.add_(d, alpha=-lr)
    if p_out is not None:
        p_out.copy_(p)


def fused_adam(p, m1, m2, vmax, g, p_out, *, lr, beta1=0.9, beta2=0.999,
               eps=1e-8, wd=0.0, step=1, amsgrad=False, gscale=1.0):
    if _require_ext(p):
        _EXT.fused_adam(p, m1, m2, vmax, g, p_out, lr, beta1, beta2, eps, wd,
                        int(step), bool(amsgrad), gscale)
        return
    d = g * gscale
    if wd != 0.0:
        d = d.add(p, alpha=wd)
    m1.mul_(beta1).add_(d, alpha=1.0 - beta1)
    m2.mul_(beta2).addcmul_(d, d, value=1.0 - beta2)
    bc1 = 1.0 - beta1 ** step
    bc2 = 1.0 - beta2 ** step
    v = m2
    if amsgrad:
        torch.maximum(vmax, m2, out=vmax)
        v = vmax
    denom = (v.sqrt() / (bc2 ** 0.5)).add_(eps)
    p.addcdiv_(m1, denom, value=-(lr / bc1))
    if p_out is not None:
        p_out.copy_(p)


# ---------------------------------------------------------------------------
# AdamW over a packed set of tensors, states in 32 or 8 bits
# ---------------------------------------------------------------------------

ACHUNK = 256  # elements that share one decay factor and one 8-bit maximum
_MASK32 = 0xffffffff


def _chunks(n: int) -> int:
    return (n + ACHUNK - 1) // ACHUNK


class State8:
    """A flat optimizer state in 8 bits: one code an element, one fp32 maximum
    for each 256 elements.

    Code k in 1..top stands for ``max * 2**((k - top) / 8)``, 0 for zero.
    ``signed=True`` (first moment): bit 7 is the sign, top is 127.
    ``signed=False`` (second moment, never negative): top is 255.
    """

    def __init__(self, codes, scales, signed):
        if codes.dtype != torch.uint8 or codes.dim() != 1:
            raise ValueError("State8 codes must be a flat uint8 tensor")
        if scales.dtype != torch.float32 or scales.dim() != 1:
            raise ValueError("State8 scales must be a flat float32 tensor")
        if scales.numel() != _chunks(codes.numel()):
            raise ValueError(
                f"State8 of {codes.numel()} elements needs "
                f"{_chunks(codes.numel())} scales, got {scales.numel()}")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("State8 tensors must be contiguous")
        if codes.device != scales.device:
            raise ValueError("State8 tensors must be on one device")
        self.codes, self.scales, self.signed = codes, scales, bool(signed)

    @classmethod
    def zeros(cls, n, signed, device=None):
        return cls(torch.zeros(n, dtype=torch.uint8, device=device),
                   torch.zeros(_chunks(n), device=device), signed)

    def span(self, start, end):
        """State8 of elements [start, end), sharing storage."""
        if not 0 <= start <= end <= self.codes.numel():
            raise ValueError(f"span [{start}, {end}) of a state of "
                             f"{self.codes.numel()} elements")
        if start % ACHUNK:
            raise ValueError(f"a span starts at a multiple of {ACHUNK}")
        if end % ACHUNK and end != self.codes.numel():
            raise ValueError(f"a span ends at a multiple of {ACHUNK} or at "
                             "the state's end")
        return State8(self.codes[start:end],
                      self.scales[start // ACHUNK:_chunks(end)], self.signed)

    def values(self, dtype=torch.float32):
        """What the codes stand for, as a new flat tensor."""
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("State8 values come as float32 or bfloat16")
        n = self.codes.numel()
        if _require_ext(self.codes):
            out = torch.empty(n, dtype=dtype, device=self.codes.device)
            _EXT.state8_values(self.codes, self.scales, out, self.signed)
            return out
        top = 127 if self.signed else 255
        c = self.codes.int()
        k = c & top
        x = torch.exp2((k - top).float() / 8)
        x = torch.where(k == 0, torch.zeros_like(x), x)
        x = x * self.scales.repeat_interleave(ACHUNK)[:n]
        return torch.where(c > top, -x, x).to(dtype)


def _overlap(written, read):
    """Whether a written tensor shares memory with another one."""
    spans = []
    for i, t in enumerate((*written, *read)):
        start = t.data_ptr()
        spans.append((start, start + t.numel() * t.element_size(),
                      i < len(written)))
    spans.sort()
    end, end_written = 0, 0   # of all so far, of those that are written
    for start, stop, w in spans:
        if start < stop:
            if start < (end if w else end_written):
                return True
            end = max(end, stop)
            end_written = max(end_written, stop) if w else end_written
    return False


def _mix32(h):
    h = h ^ (h >> 16)
    h = (h * 0x7feb352d) & _MASK32
    h = h ^ (h >> 15)
    h = (h * 0x846ca68b) & _MASK32
    return h ^ (h >> 16)


def _state8_store(st, x, r16):
    """Encode x (fp32) into st; r16 holds 16 random bits an element."""
    n, nc = x.numel(), st.scales.numel()
    top = 127 if st.signed else 255
    pad = torch.zeros(nc * ACHUNK, dtype=torch.float32, device=x.device)
    pad[:n] = x
    a = pad.view(nc, ACHUNK).abs()
    s = a.amax(1)
    s = torch.where(torch.isfinite(s), s, torch.full_like(s, float("nan")))
    e = top + 8 * torch.log2(
        a / torch.where(s > 0, s, torch.ones_like(s))[:, None])
    lo = e.floor()
    u = torch.zeros(nc * ACHUNK, dtype=torch.float32, device=x.device)
    u[:n] = (r16.float() + 0.5) / 65536
    u = u.view(nc, ACHUNK)
    up = torch.expm1((e - lo) * (math.log(2.0) / 8)) / (2 ** 0.125 - 1)
    k = (lo + (u < up)).clamp(max=top)
    if st.signed:
        low = (u < torch.exp2((e - 1) / 8)).float()
    else:
        low = torch.ones_like(e)
    k = torch.where(e < 1, low, k)
    k = torch.where(a > 0, k, torch.zeros_like(k)).nan_to_num(0.0)
    if st.signed:
        k = k + 128 * ((pad.view(nc, ACHUNK) < 0) & (k > 0))
    st.codes.copy_(k.to(torch.uint8).view(-1)[:n])
    st.scales.copy_(s)


def fused_adamw(p, m1, m2, g, p_out=None, *, lr, beta1=0.9, beta2=0.999,
                eps=1e-8, wd=0.01, step=1, gscale=1.0, decay=None, offset=0,
                seed=0):
    """One AdamW step (decoupled decay, torch.optim.AdamW's formula) in place
    over a packed set of tensors.

    p, g : flat fp32.  p_out : optional bf16/fp32 model copy.
    m1, m2 : both flat fp32, or both State8 (signed / unsigned).
    None of p, p_out and the states may share memory with another tensor.
    decay : optional fp32 factor on ``wd`` for each 256 elements (tensors that
        start at multiples of 256 get their own; None decays everything).
    offset, seed : with 8-bit states a value between two codes is rounded up
        with the probability that keeps its mean, from bits that depend on
        (offset + element index, seed, step) alone: a buffer updated in parts
        (``offset`` = where the part starts) rounds as it would in one.
        An infinity or NaN in one of the states makes that state's values of
        its 256 elements read as NaN.
    step : counts from 1; it enters as a number, so a captured graph repeats
        the step that it was captured with.
    """
    n = p.numel()
    eight = isinstance(m1, State8)
    if eight != isinstance(m2, State8):
        raise ValueError("m1 and m2 must both be fp32 or both State8")
    if eight and not (m1.signed and not m2.signed):
        raise ValueError("m1 is a signed State8, m2 an unsigned one")
    step, offset = int(step), int(offset)
    if step < 1:
        raise ValueError("step counts from 1")
    if offset < 0 or (eight and offset % ACHUNK):
        raise ValueError(f"offset must be a multiple of {ACHUNK}, 0 or more")
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError("betas must be in [0, 1)")
    flat = [("p", p), ("g", g)]
    flat += [] if eight else [("m1", m1), ("m2", m2)]
    for name, t in flat:
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32")
        if t.numel() != n:
            raise ValueError(f"{name} has {t.numel()} elements, p has {n}")
    if eight and not (m1.codes.numel() == m2.codes.numel() == n):
        raise ValueError("state and parameter lengths differ")
    if decay is not None and (decay.dtype != torch.float32
                              or not decay.is_contiguous()
                              or decay.numel() != _chunks(n)):
        raise ValueError(f"decay must be {_chunks(n)} contiguous float32 "
                         "factors, one for each 256 elements")
    if p_out is not None and (p_out.dtype not in (torch.float32,
                                                  torch.bfloat16)
                              or p_out.numel() != n
                              or not p_out.is_contiguous()):
        raise ValueError("p_out must be contiguous bf16/fp32 of p's length")
    every = [t for _, t in flat[1:]] + [t for t in (p_out, decay)
                                        if t is not None]
    every += [m1.codes, m2.codes] if eight else []
    if any(t.device != p.device for t in every):
        raise ValueError("all tensors of fused_adamw must be on one device")
    key = (int(seed) + 0x9e3779b9 * step) & _MASK32
    bc1, bc2 = 1.0 - beta1 ** step, 1.0 - beta2 ** step
    if _require_ext(p):
        _EXT.fused_adamw(p, p_out, g, m1.codes if eight else m1,
                         m2.codes if eight else m2,
                         m1.scales if eight else None,
                         m2.scales if eight else None, decay, offset,
                         lr / bc1, lr * wd, beta1, beta2, bc2 ** -0.5, eps,
                         gscale, key)
        return
    written = [p] + ([m1.codes, m1.scales, m2.codes, m2.scales] if eight
                     else [m1, m2]) + ([] if p_out is None else [p_out])
    if _overlap(written, [g] if decay is None else [g, decay]):
        raise ValueError("p, p_out and the states must not share memory with "
                         "each other, g or decay")
    d = g * gscale
    m = beta1 * (m1.values() if eight else m1) + (1.0 - beta1) * d
    v = beta2 * (m2.values() if eight else m2) + (1.0 - beta2) * d * d
    if decay is None:
        p.mul_(1.0 - lr * wd)
    else:
        p.sub_(p * (lr * wd * decay).repeat_interleave(ACHUNK)[:n])
    p.addcdiv_(m, (v.sqrt() * bc2 ** -0.5).add_(eps), value=-(lr / bc1))
    if p_out is not None:
        p_out.copy_(p)
    if eight:
        i = torch.arange(offset, offset + n, device=p.device)
        r = _mix32((i & _MASK32) ^ _mix32((key + (i >> 32)) & _MASK32))
        _state8_store(m1, m, r & 0xffff)
        _state8_store(m2, v, r >> 16)
    else:
        m1.copy_(m)
        m2.copy_(v)


# ---------------------------------------------------------------------------
# dense multi-source reduction (deterministic source order)
# ---------------------------------------------------------------------------

def reduce_accum(dst, srcs, scale=1.0, beta=0.0):
    """dst(f32) = beta*dst + scale * sum_r srcs[r]  (srcs all bf16 or all f32).

    Any source count: the kernel takes 8 sources per launch (PtrPack), so
    longer lists chunk into passes accumulating with beta=1 — no world-size
    cliff."""
    srcs = list(srcs)
    if _require_ext(dst):
        for i in range(0, len(srcs), 8):
            _EXT.reduce_accum(dst, srcs[i:i + 8], scale,
                              beta if i == 0 else 1.0)
        return
    acc = torch.zeros_like(dst)
    for s in srcs:
        acc += s.float()
    if beta == 0.0:
        dst.copy_(acc * scale)
    else:
        dst.mul_(beta).add_(acc, alpha=scale)


def f32_to_bf16(src, dst):
    if _require_ext(src):
        _EXT.f32_to_bf16(src, dst)
        return
    dst.copy_(src)


def bf16_to_f32(src, dst):
    if _require_ext(dst):
        _EXT.bf16_to_f32(src, dst)
        return
    dst.copy_(src)


# ---------------------------------------------------------------------------
# int8 gradient quantization (per-256-element absmax chunks)
# ---------------------------------------------------------------------------

def quant8_nscales(n: int) -> int:
    return (n + QCHUNK - 1) // QCHUNK


def quant8_encode(src, scales, q):
    if _require_ext(src):
        _EXT.quant8_encode(src, scales, q)
        return
    n = src.numel()
    nc = quant8_nscales(n)
    pad = nc * QCHUNK - n
    x = src.float()
    if pad:
        x = torch.cat([x, x.new_zeros(pad)])
    x = x.view(nc, QCHUNK)
    absmax = x.abs().amax(dim=1)
    s = torch.where(absmax > 0, absmax / 127.0, torch.ones_like(absmax))
    scales[:nc].copy_(s)
    qv = torch.clamp(torch.round(x / s[:, None]), -127, 127).to(torch.int8)
    q[:n].copy_(qv.view(-1)[:n])


def quant8_reduce(dst, scales_list, qs_list, gscale=1.0, beta=0.0):
    """Any source count (8 per kernel pass, accumulated — see reduce_accum)."""
    scales_list = list(scales_list)
    qs_list = list(qs_list)
    if _require_ext(dst):
        for i in range(0, len(qs_list), 8):
            _EXT.quant8_reduce(dst, scales_list[i:i + 8], qs_list[i:i + 8],
                               gscale, beta if i == 0 else 1.0)
        return
    n = dst.numel()
    acc = torch.zeros_like(dst)
    for s, q in zip(scales_list, qs_list):
        sc = s.repeat_interleave(QCHUNK)[:n]
        acc += sc * q[:n].float()
    if beta == 0.0:
        dst.copy_(acc * gscale)
    else:
        dst.mul_(beta).add_(acc, alpha=gscale)


# ---------------------------------------------------------------------------
# top-k magnitude sparsification
# ---------------------------------------------------------------------------

def topk_workspace(device) -> torch.Tensor:
    return torch.zeros(TOPK_WS_WORDS, dtype=torch.int32, device=device)


def topk_encode(src, k, ws, out_idx, out_val):
    """Select k largest-|x| elements -> (out_idx int32, out_val src.dtype).

    GPU: radix-style bin threshold (ties within the boundary bin are taken in
    arbitrary order).  CPU: exact torch.topk.
    """
    if _require_ext(src):
        _EXT.topk_encode(src, int(k), ws, out_idx, out_val)
        return
    v, idx = torch.topk(src.float().abs(), int(k), sorted=False)
    out_idx[:k].copy_(idx.to(torch.int32))
    out_val[:k].copy_(src[idx])


def topk_scatter(dst, idx, val, k, gscale=1.0):
    """dst[idx[:k]] += gscale * val[:k] — one message (unique indices)."""
    if _require_ext(dst):
        _EXT.topk_scatter(dst, idx, val, int(k), gscale)
        return
    dst.index_add_(0, idx[:k].long(), val[:k].float() * gscale)


def _keys_of(x):
    """11-bit magnitude key: float32 bits of |x| >> 21 (matches tk_key)."""
    return (x.float().abs().contiguous().view(torch.int32) >> 21) & 0x7FF


def topk_thresh_encode(src, off_keys, kmax, ws, hdr, out_idx, out_val):
    """VARIABLE-k selection: every element within `off_keys` magnitude-key
    steps (1/8 octave each) of the bucket's peak |x|, capped at kmax;
    k_used lands in the int32 `hdr` — the device-side variable-length wire
    (the reference's adaptive codecs sized payloads by content).
    """
    if _require_ext(src):
        _EXT.topk_encode_thresh(src, int(off_keys), int(kmax), ws, hdr,
                                out_idx, out_val)
        return
    keys = _keys_of(src)
    thr0 = max(0, int(keys.max()) - int(off_keys))
    cand = int((keys >= thr0).sum())
    k = max(1, min(cand, int(kmax)))
    v, idx = torch.topk(src.float().abs(), k, sorted=False)
    hdr[0] = k
    out_idx[:k].copy_(idx.to(torch.int32))
    out_val[:k].copy_(src[idx])


def topk_scatter_var(dst, hdr, idx, val, kmax, gscale=1.0):
    """dst[idx[:k]] += gscale * val[:k] with k read from the device header."""
    if _require_ext(dst):
        _EXT.topk_scatter_var(dst, hdr, idx, val, int(kmax), gscale)
        return
    k = int(hdr[0])
    dst.index_add_(0, idx[:k].long(), val[:k].float() * gscale)


from . import bn  # noqa: E402,F401  (fused BatchNorm module; needs ops ready)
from . import ln  # noqa: E402,F401
from . import ce  # noqa: E402,F401
from . import attn  # noqa: E402,F401
from . import linear  # noqa: E402,F401
from . import rope  # noqa: E402,F401
