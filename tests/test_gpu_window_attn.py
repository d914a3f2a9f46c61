"""Sliding-window attention kernels against 64 bits (@gpu).

Bounds, element by element.  e = 2^-8 is half a step of bf16; P and dS are
rounded to bf16 as operands of the products, sums are fp32.
  o:  e |o| + e sum_j P_ij |v_j|
  delta (rowsum(dO * o), o rounded): e sum_d |dO o|
  dS: e |dS| + P * (delta's error), and so on through dQ, dK
with S = 2^-15 of the magnitudes for fp32 scores of 64 to 128 products, their
exponentials and sums.
"""

import pytest
import torch

from pytorch_ps_mpi_amd.ops import attn
from pytorch_ps_mpi_amd.ops.attn import fused_window_sdpa
from test_window_attn import by_hand

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E, S = 2.0 ** -8, 2.0 ** -15


def _bounds(q, k, v, go, window, sinks, lengths, scale, want):
    B, H, N, D = q.shape
    G = H // k.shape[1]
    q, k, v, go = (t.double().to(DEV) for t in (q, k, v, go))
    o, dq, dk, dv = (t.to(DEV) for t in want)
    to, tq = E * o.abs(), E * dq.abs()
    tk, tv = E * dk.abs(), E * dv.abs()
    for b in range(B):
        n = N if lengths is None else max(0, min(N, int(lengths[b])))
        if n == 0:
            continue
        i = torch.arange(n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None]
        vis = (j <= i) & ((i - j < window) | (j < sinks))
        for h in range(H):
            g = h // G
            Q, K, V, R = q[b, h, :n], k[b, g, :n], v[b, g, :n], go[b, h, :n]
            O = o[b, h, :n]
            Kt, Vt = K.t().contiguous(), V.t().contiguous()
            P = torch.softmax((Q @ Kt * scale).masked_fill(~vis, -torch.inf),
                              1)
            # a score's fp32 error moves its weight by that part
            rel = S * (1 + (Q.abs() @ Kt.abs() * scale))
            eP = P * rel
            to[b, h, :n] += (E * P + eP) @ V.abs()
            dP = R @ Vt
            ddel = (R * O).abs().sum(1, keepdim=True)
            dd = dP - (R * O).sum(1, keepdim=True)
            dS = P * dd
            edd = (E + S) * ddel + S * (R.abs() @ Vt.abs())
            eS = (E * dS.abs() + eP * dd.abs() + P * edd) * scale
            tq[b, h, :n] += eS @ K.abs()
            tk[b, g, :n] += eS.t().contiguous() @ Q.abs()
            tv[b, g, :n] += (E * P + eP).t().contiguous() @ R.abs()
    return [t.cpu() for t in (to, tq, tk, tv)]


def _make(B, H, KV, N, D, seed=0, peak=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda h, s=1.0: (torch.randn(B, h, N, D, generator=g) * s).bfloat16()  # noqa: E731
    return mk(H, peak), mk(KV), mk(KV), mk(H)


def _check(q, k, v, go, window, sinks, lengths=None, scale=None, dev=None):
    D = q.shape[3]
    want = by_hand(q, k, v, go, window, sinks, lengths, scale or D ** -0.5)
    tol = _bounds(q, k, v, go, window, sinks, lengths, scale or D ** -0.5,
                  want)
    dq, dk, dv, dgo = dev or [t.to(DEV) for t in (q, k, v, go)]
    leaves = [t.detach().requires_grad_() for t in (dq, dk, dv)]
    lens = None if lengths is None else lengths.to(DEV)
    o = fused_window_sdpa(*leaves, window, sinks, lens, scale)
    got = (o.detach(), *torch.autograd.grad(o, leaves, dgo))
    for name, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, tol):
        assert a.shape == b.shape and a.dtype == torch.bfloat16
        err = (a.cpu().double() - b).abs()
        assert (err <= t + 1e-30).all(), (name, err.max(), (err / t).max())
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129,
                               200, 300])
def test_lengths_of_a_sequence(D, N):
    _check(*_make(1, 2, 2, N, D, N), window=40, sinks=3)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [
    (1, 0), (1, 1), (2, 500), (31, 0), (32, 1), (33, 32), (64, 64), (65, 33),
    (100, 130), (128, 0), (299, 4), (300, 0), (10 ** 6, 10 ** 6), (7, 129),
])
def test_windows_and_sinks(D, window, sinks):
    _check(*_make(1, 1, 1, 300, D, window), window=window, sinks=sinks)


@pytest.mark.parametrize("H,KV", [(1, 1), (3, 3), (6, 2), (4, 1), (8, 2),
                                  (10, 2), (16, 1), (6, 1)])
def test_head_groups(H, KV):
    _check(*_make(2, H, KV, 150, 64, H), window=50, sinks=2)


@pytest.mark.parametrize("B,H,KV,N,D,window,sinks", [
    (4, 64, 64, 257, 64, 60, 5),      # key blocks for more than two rounds
    (4, 64, 64, 257, 128, 60, 0),
    (6, 32, 16, 300, 64, 50, 130),    # more than one round, first tokens
    (1, 8, 1, 1500, 64, 100, 200),    # few key blocks: their rows shared out
    (2, 6, 1, 700, 128, 90, 33),
])
def test_how_blocks_share_the_work(B, H, KV, N, D, window, sinks):
    _check(*_make(B, H, KV, N, D, N), window=window, sinks=sinks)


@pytest.mark.parametrize("D", [64, 128])
def test_padded_batches(D):
    """Lengths zero, one, odd, whole, and beyond the tensor; what stands behind
    a length is NaN or infinite and is neither read nor passed on."""
    B, N = 6, 170
    q, k, v, go = _make(B, 4, 2, N, D, 5)
    lengths = torch.tensor([0, 1, 65, 169, 170, 999], dtype=torch.int32)
    clean = [t.clone() for t in (q, k, v, go)]
    for b, n in enumerate(lengths.tolist()):
        for t, bad in zip((q, k, v, go), (torch.nan, torch.inf, -torch.inf,
                                          torch.nan)):
            t[b, :, n:] = bad
        for t in clean:
            t[b, :, n:] = 0
    got = _check(*clean, 40, 3, lengths, dev=[t.to(DEV)
                                              for t in (q, k, v, go)])
    for t in got:
        for b, n in enumerate(lengths.tolist()):
            assert (t[b, :, n:] == 0).all()


@pytest.mark.parametrize("peak", [8.0, 30.0])
def test_peaked_scores(peak):
    """Scores of some hundred: the running maximum jumps late, most weights
    are zero."""
    q, k, v, go = _make(1, 2, 1, 200, 64, 7, peak)
    k[:, :, 150] *= 4
    _check(q, k, v, go, 80, 5)


def test_scale():
    _check(*_make(1, 2, 2, 90, 64, 8), window=33, sinks=1, scale=0.01)


def test_long_sequence_with_sinks():
    """Rows far behind the window see the first tokens alone: their gradients
    come from all parts of the sequence."""
    _check(*_make(1, 2, 1, 2500, 64, 9), window=70, sinks=130)
    _check(*_make(1, 1, 1, 1500, 128, 9), window=200, sinks=4)


def test_strides():
    """Slices of a fused projection, heads behind rows, expanded batches, odd
    offsets, gradients of another layout: all the same numbers."""
    B, H, KV, N, D = 2, 4, 2, 100, 64
    q, k, v, go = (t.to(DEV) for t in _make(B, H, KV, N, D, 10))

    def run(q, k, v, go):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        o = fused_window_sdpa(*x, 30, 2)
        return [o.detach(), *torch.autograd.grad(o, x, go)]

    want = run(q, k, v, go)
    fused = torch.cat([t.transpose(1, 2) for t in (q, k, v)], 2)
    parts = [t.transpose(1, 2) for t in fused.split([H, KV, KV], 2)]
    behind = go.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(k.numel() + 1, dtype=k.dtype, device=DEV)
    odd[1:] = k.reshape(-1)
    wide = torch.zeros(B, KV, N, 2 * D, dtype=k.dtype, device=DEV)
    wide[..., ::2] = v
    for args in ((*parts, go), (q, k, v, behind),
                 (q, odd[1:].view(k.shape), wide[..., ::2], go)):
        for a, b in zip(run(*args), want):
            assert torch.equal(a, b)
    one = run(q[:1].expand(B, -1, -1, -1), k, v, go)
    two = run(q[:1].repeat(B, 1, 1, 1), k, v, go)
    for a, b in zip(one, two):
        assert torch.equal(a, b)
    # a gradient that is one number for all: no strides at all
    same = torch.full((), 0.5, device=DEV, dtype=torch.bfloat16)
    a = run(q, k, v, same.expand(B, H, N, D))
    b = run(q, k, v, same.expand(B, H, N, D).contiguous())
    for s, t in zip(a, b):
        assert torch.equal(s, t)


def test_repeats_streams_and_graphs():
    q, k, v, go = (t.to(DEV) for t in _make(2, 8, 2, 700, 64, 11))
    lens = torch.tensor([700, 333], dtype=torch.int32, device=DEV)
    x = [t.detach().requires_grad_() for t in (q, k, v)]

    def step():
        o = fused_window_sdpa(*x, 90, 4, lens)
        g = torch.autograd.grad(o, x, go)
        return [o.detach(), *g]

    want = step()
    for a, b in zip(step(), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x[1].mul_(0.9)
            lens[0] -= 100
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_types_without_kernel_and_refusals():
    q, k, v, go = (t.to(DEV) for t in _make(1, 2, 1, 40, 64, 12))
    want = fused_window_sdpa(q, k, v, 9, 2).double()
    o32 = fused_window_sdpa(q.float(), k.float(), v.float(), 9, 2)
    assert (want - o32.double()).norm() <= 2 * E * want.norm()
    o = fused_window_sdpa(q[..., :48], k[..., :48], v[..., :48], 9, 2)
    assert o.shape == (1, 2, 40, 48)
    e = torch.empty(0, 2, 5, 64, dtype=torch.bfloat16, device=DEV)
    assert fused_window_sdpa(e, e, e, 3).shape == e.shape
    with pytest.raises(ValueError):
        fused_window_sdpa(q, k.cpu(), v, 9)
    with pytest.raises(ValueError):
        fused_window_sdpa(q, k, v, 9, lengths=torch.tensor([3],
                                                           dtype=torch.int32))
    with pytest.raises(RuntimeError):  # the extension checks for itself
        attn._EXT.window_sdpa(q, k, v[:, :, :9], 9, 0, None, 1.0)
    x = q.detach().requires_grad_()
    o = fused_window_sdpa(x, k, v, 9)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(o.sum(), x, create_graph=True)


def test_more_first_tokens_than_a_launch_holds():
    """Sums of 2^21 first tokens over all key heads are one launch; the last
    heads' take another.  The first and the last heads against 64 bits."""
    H, N, window, sinks = 520, 4100, 2, 4097
    assert H * sinks > 2 ** 21
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, v, go = (torch.randn(1, H, N, 64, generator=g, device=DEV).bfloat16()
                   for _ in range(4))
    x = [t.requires_grad_() for t in (q, k, v)]
    o = fused_window_sdpa(*x, window, sinks)
    got = (o.detach(), *torch.autograd.grad(o, x, go))
    for h in (0, H - 1):
        part = [t.detach()[:, h:h + 1].cpu() for t in (q, k, v, go)]
        want = by_hand(*part, window, sinks, None, 0.125)
        tol = _bounds(*part, window, sinks, None, 0.125, want)
        for name, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, tol):
            err = (a[:, h:h + 1].cpu().double() - b).abs()
            assert (err <= t + 1e-30).all(), (h, name, err.max())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks,lengths", [
    (2, 0, None), (5, 1, None), (40, 0, [150, 61]),
])
def test_gradients_of_values_with_a_common_part(D, window, sinks, lengths):
    """dS = P * (dP - rowsum(dO * O)): a part that all values share cancels.
    With O rounded to bf16 in that sum its error would not: what the rounding
    left out is kept, itself rounded, so the sum is off by E * E of its
    magnitude and the fp32 part S.  O's weights P' are rounded for their product
    and divided by their own sum: |P' - P| <= 2 E P, and as both add up to 1
    the sum is off by |sum_j (P' - P)(dP - delta)| <= 2 E sum_j P |dP - delta|,
    whatever the values share.  The other terms are as in _bounds."""
    B, H, N = 2, 2, 150
    q, k, v, go = _make(B, H, 1, N, D, 21)
    v = (v.float() + 6.0).bfloat16()
    lens = None if lengths is None else torch.tensor(lengths,
                                                     dtype=torch.int32)
    scale = D ** -0.5
    want = by_hand(q, k, v, go, window, sinks, lens, scale)
    x = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    o = fused_window_sdpa(*x, window, sinks,
                          None if lens is None else lens.to(DEV))
    dq, dk, _ = torch.autograd.grad(o, x, go.to(DEV))
    tq, tk = E * want[1].abs(), E * want[2].abs()
    for b in range(B):
        n = N if lens is None else int(lens[b])
        i, j = torch.arange(n)[:, None], torch.arange(n)[None]
        vis = (j <= i) & ((i - j < window) | (j < sinks))
        K, V = k[b, 0, :n].double(), v[b, 0, :n].double()
        for h in range(H):
            Q, R = q[b, h, :n].double(), go[b, h, :n].double()
            P = torch.softmax((Q @ K.t() * scale).masked_fill(
                ~vis, -torch.inf), 1)
            eP = P * S * (1 + (Q.abs() @ K.t().abs() * scale))
            # P's own fp32 error moves O and with it the sum
            O = P @ V
            dd = R @ V.t() - (R * O).sum(1, keepdim=True)
            edd = (E * E + S) * (R * O).abs().sum(1, keepdim=True) \
                + S * (R.abs() @ V.t().abs()) \
                + 2 * E * (P * dd).abs().sum(1, keepdim=True)
            eS = (E * (P * dd).abs() + eP * dd.abs() + P * edd) * scale
            tq[b, h, :n] += eS @ K.abs()
            tk[b, 0, :n] += eS.t() @ Q.abs()
    for name, a, w, t in (("dq", dq, want[1], tq), ("dk", dk, want[2], tk)):
        err = (a.cpu().double() - w).abs()
        assert (err <= t + 1e-30).all(), (name, err.max(), (err / t).max())
