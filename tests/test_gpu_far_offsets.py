"""The transformer-step operators on tensors of more than 2^31 elements (@gpu):
what lies behind that must be what a call on the end alone gives.  Each test
holds 20 to 45 GB."""

import pytest
import torch

from pytorch_ps_mpi_amd import ops
from pytorch_ps_mpi_amd.ops.attn import fused_window_sdpa
from pytorch_ps_mpi_amd.ops.ln import fused_gated_residual
from pytorch_ps_mpi_amd.ops.rope import AxialRotary
from test_gpu_window_attn import _bounds
from test_window_attn import by_hand

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _randn(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.bfloat16)


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def test_window_attention():
    """A sequence whose last rows see the first token and their window: a
    short one of that token and the last 400 gives the same rows, and the same
    gradients of keys that only those rows see."""
    H, N, D, window = 64, 270_000, 128, 32
    x = [_randn(1, N, H, D, seed=s).transpose(1, 2).requires_grad_()
         for s in range(3)]
    go = _randn(1, N, H, D, seed=3).transpose(1, 2)
    assert x[0].numel() > 2 ** 31
    o = fused_window_sdpa(*x, window, 1)
    got = (o.detach(), *torch.autograd.grad(o, x, go))
    at = torch.cat([torch.zeros(1, dtype=torch.long),
                    torch.arange(N - 400, N)]).to(DEV)
    for h in (0, H - 1):
        part = [t.detach()[:, h:h + 1, at].cpu() for t in (*x, go)]
        want = by_hand(*part, window, 1, None, D ** -0.5)
        tol = _bounds(*part, window, 1, None, D ** -0.5, want)
        for name, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, tol):
            a = a[:, h:h + 1, at].cpu().double()
            err = (a - b).abs()[:, :, -300:]
            assert (err <= t[:, :, -300:] + 1e-30).all(), (h, name, err.max())


def test_gated_residual():
    rows, D = 1_200_000, 2048
    x, u, gy, gh = (_randn(rows, D, seed=s) for s in range(4))
    w, gate = _randn(D, seed=4), _randn(D, seed=5)
    assert x.numel() > 2 ** 31

    def run(part):
        t = [v[part].requires_grad_() for v in (x, u)]
        y, h = fused_gated_residual(*t, w, gate=gate)
        g = torch.autograd.grad((y, h), t, (gy[part], gh[part]))
        return [v.detach()[-5:].clone() for v in (y, h, *g)]

    for a, b in zip(run(slice(None)), run(slice(rows - 5, rows))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(interleaved):
    N, H, D = 1_500_000, 12, 128
    q, k = (_randn(1, N, H, D, seed=s) for s in range(2))
    pos = torch.stack([torch.arange(N, device=DEV),
                       torch.arange(N, device=DEV) % 1000])
    rot = AxialRotary(D, (40, 24), interleaved=interleaved)
    assert q.numel() > 2 ** 31
    whole = [t[:, -7:].clone() for t in rot(q, k, pos)]
    for a, b in zip(whole, rot(q[:, -7:], k[:, -7:], pos[:, -7:])):
        assert torch.equal(a, b)


def test_adamw():
    """More than 2^32 elements in 8 bits: the end as a part with its offset."""
    n = 2 ** 32 + 777
    start = 2 ** 32 - 512
    p = torch.zeros(n, device=DEV)
    g = torch.zeros(n, device=DEV)
    g[start:] = _randn(n - start).float()
    g[:512] = 1.0
    m, v = ops.State8.zeros(n, True, DEV), ops.State8.zeros(n, False, DEV)
    pe = p[start:].clone()
    me, ve = (ops.State8.zeros(n - start, s, DEV) for s in (True, False))
    for step in (1, 2):
        ops.fused_adamw(p, m, v, g, lr=1e-2, step=step, seed=3)
        ops.fused_adamw(pe, me, ve, g[start:].clone(), lr=1e-2, step=step,
                        seed=3, offset=start)
    assert torch.equal(p[start:], pe) and pe.abs().min() > 0
    for a, b in ((m, me), (v, ve)):
        assert torch.equal(a.codes[start:], b.codes)
        assert torch.equal(a.scales[start // 256:], b.scales)
        assert torch.equal(a.values()[start:], b.values())
    assert not p[512:start].any()
