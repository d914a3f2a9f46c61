"""Sliding-window attention with visible first tokens: CPU path, refusals."""

import math

import pytest
import torch

from pytorch_ps_mpi_amd.ops.attn import fused_window_sdpa


def by_hand(q, k, v, go, window, sinks, lengths, scale):
    """64-bit o, dq, dk, dv, one sequence and head at a time."""
    B, H, N, D = q.shape
    G = H // k.shape[1]
    q, k, v, go = (t.double() for t in (q, k, v, go))
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    for b in range(B):
        n = N if lengths is None else max(0, min(N, int(lengths[b])))
        if n == 0:
            continue
        i, j = torch.arange(n)[:, None], torch.arange(n)[None]
        vis = (j <= i) & ((i - j < window) | (j < sinks))
        for h in range(H):
            g = h // G
            Q, K, V, R = q[b, h, :n], k[b, g, :n], v[b, g, :n], go[b, h, :n]
            P = torch.softmax((Q @ K.t() * scale).masked_fill(~vis, -math.inf),
                              1)
            O = P @ V
            dS = P * (R @ V.t() - (R * O).sum(1, keepdim=True)) * scale
            o[b, h, :n], dq[b, h, :n] = O, dS @ K
            dk[b, g, :n] += dS.t() @ Q
            dv[b, g, :n] += P.t() @ R
    return o, dq, dk, dv


@pytest.mark.parametrize("B,H,KV,N,D,window,sinks,lengths", [
    (1, 1, 1, 1, 4, 1, 0, None), (2, 4, 2, 7, 8, 3, 1, None),
    (1, 2, 1, 9, 5, 1, 0, None), (2, 3, 3, 6, 8, 100, 100, None),
    (3, 2, 1, 8, 4, 2, 2, [8, 0, 3]),
])
def test_cpu_against_definition(B, H, KV, N, D, window, sinks, lengths):
    g = torch.Generator().manual_seed(0)
    q = torch.randn(B, H, N, D, generator=g, requires_grad=True)
    k, v = (torch.randn(B, KV, N, D, generator=g, requires_grad=True)
            for _ in range(2))
    go = torch.randn(B, H, N, D, generator=g)
    lens = None if lengths is None else torch.tensor(lengths,
                                                     dtype=torch.int32)
    o = fused_window_sdpa(q, k, v, window, sinks, lens)
    got = (o.detach(), *torch.autograd.grad(o, (q, k, v), go))
    want = by_hand(q.detach(), k.detach(), v.detach(), go, window, sinks,
                   lens, D ** -0.5)
    for a, b in zip(got, want):
        assert torch.allclose(a.double(), b, atol=1e-5)


def test_cpu_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(1, 2, 5, 3, generator=g, dtype=torch.float64)
    k, v = (torch.randn(1, 1, 5, 3, generator=g, dtype=torch.float64)
            for _ in range(2))
    assert torch.autograd.gradcheck(
        lambda a, b, c: fused_window_sdpa(a, b, c, 2, 1),
        [t.requires_grad_() for t in (q, k, v)])


def test_wide_window_is_causal_attention():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(2, 3, 10, 8, generator=g) for _ in range(3))
    want = torch.nn.functional.scaled_dot_product_attention(q, k, v,
                                                            is_causal=True)
    assert torch.allclose(fused_window_sdpa(q, k, v, 10), want, atol=1e-5)


def test_refusals():
    q, k = torch.zeros(2, 4, 6, 8), torch.zeros(2, 2, 6, 8)
    n = torch.tensor([6, 2], dtype=torch.int32)
    fused_window_sdpa(q, k, k, 3, 1, n)
    bad = [
        ((q[0], k, k, 3), {}), ((q, k, k[:, :1], 3), {}),
        ((q, k[:, :, :5], k[:, :, :5], 3), {}),
        ((q[:, :3], k, k, 3), {}), ((q, k[..., :4], k[..., :4], 3), {}),
        ((q[:1], k, k, 3), {}), ((q.double(), k, k, 3), {}),
        ((q.int(), k.int(), k.int(), 3), {}), ((q, k, k, 0), {}),
        ((q, k, k, 3, -1), {}), ((q, k, k, 3), dict(lengths=n.long())),
        ((q, k, k, 3), dict(lengths=n[:1])), ((q, k, k, 3), dict(scale=0.0)),
        ((q, k, k, 3), dict(scale=-1.0)),
        ((q, k, k, 3), dict(scale=math.inf)),
        ((q, k[:, :0], k[:, :0], 3), {}),
    ]
    for args, kw in bad:
        with pytest.raises(ValueError):
            fused_window_sdpa(*args, **kw)
