"""Rotary kernels against the 64-bit definition (@gpu)."""

import pytest
import torch

from pytorch_ps_mpi_amd.ops.rope import AxialRotary
from test_rope import by_hand

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _tol(x, dtype):
    """Half a step of the output, plus fp32 arithmetic: cos and sin each off
    by 2^-23 at most (a fraction of a turn rounded to 32 bits, the function),
    two products, a sum: 6 * 2^-24 of the pair's magnitude (<= 2 max)."""
    return torch.finfo(dtype).eps / 2 * x.abs() + 6 * 2 ** -24 * 2 * 6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
@pytest.mark.parametrize("B,N,H,KV,D,sections", [
    (1, 1, 1, 1, 2, (1,)), (2, 7, 3, 1, 10, (1, 2, 1)),
    (1, 5, 4, 2, 64, (16, 16)), (3, 33, 12, 12, 64, (8, 8, 8)),
    (2, 9, 8, 2, 128, (16, 24, 24)), (1, 6, 2, 1, 96, (17, 20)),
    (1, 3, 1, 1, 512, (256,)), (2, 5, 2, 2, 80, (5, 9, 7, 3)),
    (1, 4, 40, 8, 128, (31, 32)),
])
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_backward(dtype, B, N, H, KV, D, sections, interleaved):
    g = torch.Generator().manual_seed(B * 1000 + N)
    mk = lambda *s: torch.randn(*s, generator=g).clamp(-6, 6).to(dtype)  # noqa: E731
    q, k, gq, gk = (mk(B, N, h, D) for h in (H, KV, H, KV))
    pos = torch.randint(0, 2_000_000, (len(sections), B, N), generator=g)
    rot = AxialRotary(D, sections, shared=N % 2 == 0, interleaved=interleaved)
    qd, kd = (t.to(DEV).requires_grad_() for t in (q, k))
    y = rot(qd, kd, pos.to(DEV) if N % 3 else pos.to(DEV, torch.int32))
    d = torch.autograd.grad(y, (qd, kd), (gq.to(DEV), gk.to(DEV)))
    for got, x, sign in ((y[0], q, 1), (y[1], k, 1), (d[0], gq, -1),
                         (d[1], gk, -1)):
        assert got.dtype == dtype and got.shape == x.shape
        want = by_hand(x, pos, sections, N % 2 == 0, interleaved, sign=sign)
        err = (got.detach().cpu().double() - want).abs()
        assert (err <= _tol(want, dtype)).all(), err.max()


def test_strided_inputs():
    """Slices of a fused projection, transposed heads, broadcast batches and
    gradients that are views: no copy is needed and none changes the result."""
    g = torch.Generator().manual_seed(3)
    B, N, H, D = 2, 13, 4, 64
    rot = AxialRotary(D, (16, 16))
    pos = torch.randint(0, 99, (2, N), generator=g).to(DEV)
    qkv = torch.randn(B, N, 3, H, D, generator=g).bfloat16().to(DEV)
    a = rot(qkv[:, :, 0], qkv[:, :, 1], pos)
    b = rot(qkv[:, :, 0].contiguous(), qkv[:, :, 1].contiguous(),
            pos[:, None].expand(2, B, N).contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = qkv[:, :, 0].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(rot(t, t, pos)[0], b[0])
    # odd storage offset: no 16-byte alignment
    flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)
    flat[1:] = t.reshape(-1)
    o = flat[1:].view(B, N, H, D)
    assert torch.equal(rot(o, o, pos)[1], b[0])
    wide = torch.zeros(B, N, H, 2 * D, dtype=t.dtype, device=DEV)
    wide[..., ::2] = t  # last stride 2
    assert torch.equal(rot(wide[..., ::2], t, pos)[0], b[0])
    q = t.detach().requires_grad_()
    gr = torch.randn(B, H, N, D, generator=g).bfloat16().to(DEV)
    yq, _ = rot(q, t, pos)
    (d1,) = torch.autograd.grad(yq, q, gr.transpose(1, 2), retain_graph=True)
    (d2,) = torch.autograd.grad(yq, q, gr.transpose(1, 2).contiguous())
    assert torch.equal(d1, d2)


def test_empty_and_refusals():
    rot = AxialRotary(8, (2, 2))
    q = torch.zeros(0, 3, 4, 8, device=DEV)
    pos = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    assert rot(q, q, pos)[0].shape == q.shape
    q = torch.zeros(1, 3, 4, 8, device=DEV)
    with pytest.raises(ValueError):
        rot(q, q.cpu(), pos)
    with pytest.raises(ValueError):
        rot(q, q, pos.cpu())
    with pytest.raises(ValueError):
        rot(q.double(), q.double(), pos)


def test_graph_replays():
    rot = AxialRotary(64, (16, 16))
    q = torch.randn(2, 50, 4, 64, device=DEV).bfloat16()
    pos = torch.arange(50, device=DEV).expand(2, 50).contiguous()
    s = torch.cuda.CUDAGraph()
    with torch.cuda.graph(s):
        y, z = rot(q, q, pos)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        pos.add_(i)
        s.replay()
        torch.cuda.synchronize()
        want = rot(q, q, pos)
        assert torch.equal(y, want[0]) and torch.equal(z, want[1])


def test_more_rows_than_a_launch_holds():
    """2^23 blocks of four tokens are one launch; the rest take another."""
    N = 2 ** 25 + 7
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(1, N, 1, 2, generator=g, device=DEV).bfloat16()
    pos = torch.randint(0, 2_000_000, (1, N), generator=g, device=DEV,
                        dtype=torch.int32)
    rot = AxialRotary(2, (1,))
    y, _ = rot(x, x[:, :, :1], pos)
    for part in (slice(0, 50), slice(2 ** 25 - 50, N)):
        want = by_hand(x[:, part].cpu(), pos[:, None, part].cpu(), (1,), False,
                       False)
        err = (y[:, part].cpu().double() - want).abs()
        assert (err <= _tol(want, torch.bfloat16)).all(), err.max()
    assert torch.equal(y[:, 2 ** 24:], rot(x[:, 2 ** 24:], x[:, 2 ** 24:],
                                           pos[:, 2 ** 24:])[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,sections", [
    (96, (10, 6, 9)), (96, (43,)), (96, (20, 12, 12)), (64, (6, 4)),
    (64, (30,)), (64, (3,)), (128, (17, 10, 15)), (20, (8,)), (17, (8,)),
    (33, (5, 6)), (9, (4,)), (7, (1, 1)), (30, (15,)), (22, (9,)),
])
def test_ranges_that_vectors_do_not_divide(dtype, interleaved, D, sections):
    """What turns and what passes through end anywhere; the latter keeps its
    bits, NaN included, and results repeat."""
    g = torch.Generator().manual_seed(D)
    q, k = (torch.randn(2, 9, h, D, generator=g).clamp(-6, 6).to(dtype)
            for h in (5, 2))
    P = sum(sections)
    if 2 * P < D:
        q[:, ::2, :, 2 * P:] = float("nan")
        q[:, 1::2, :, -1] = float("inf")
    pos = torch.randint(0, 100_000, (len(sections), 2, 9), generator=g)
    rot = AxialRotary(D, sections, interleaved=interleaved)
    args = (q.to(DEV), k.to(DEV), pos.to(DEV))
    y = rot(*args)
    for got, x in zip(y, (q, k)):
        got = got.cpu()
        if 2 * P < D:
            bits = torch.int16 if dtype == torch.bfloat16 else torch.int32
            assert torch.equal(got[..., 2 * P:].contiguous().view(bits),
                               x[..., 2 * P:].contiguous().view(bits))
        want = by_hand(x, pos, sections, False, interleaved)[..., :2 * P]
        err = (got[..., :2 * P].double() - want).abs()
        assert (err <= _tol(want, dtype)).all(), err.max()
    for _ in range(3):
        for a, b in zip(rot(*args), y):
            assert torch.equal(a.nan_to_num(), b.nan_to_num())
