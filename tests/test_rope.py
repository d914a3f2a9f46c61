"""Rotary positions with several axes: the CPU path and its refusals."""

import math

import pytest
import torch

from pytorch_ps_mpi_amd.ops.rope import AxialRotary


def by_hand(x, pos, sections, shared, interleaved, base=10000.0, sign=1.0):
    """64-bit definition, pair by pair."""
    x, y = x.double(), x.double().clone()
    P, p = sum(sections), 0
    for a, n in enumerate(sections):
        for i in range(n):
            f = base ** (-(p / P if shared else i / n))
            t = sign * pos[a].double() * f
            c, s = torch.cos(t)[..., None], torch.sin(t)[..., None]
            ia, ib = (2 * p, 2 * p + 1) if interleaved else (p, P + p)
            y[..., ia] = x[..., ia] * c - x[..., ib] * s
            y[..., ib] = x[..., ia] * s + x[..., ib] * c
            p += 1
    return y


@pytest.mark.parametrize("D,sections", [(8, (2, 2)), (10, (1, 2, 1)),
                                        (6, (3,)), (64, (4, 3, 5, 6))])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_cpu_against_definition(D, sections, shared, interleaved):
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 5, 3, D, generator=g, requires_grad=True)
    k = torch.randn(2, 5, 1, D, generator=g, requires_grad=True)
    pos = torch.randint(0, 1 << 20, (len(sections), 2, 5), generator=g)
    rot = AxialRotary(D, sections, shared=shared, interleaved=interleaved)
    yq, yk = rot(q, k, pos)
    gq, gk = torch.randn(yq.shape, generator=g), torch.randn(yk.shape,
                                                             generator=g)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    # cos and sin rounded once, two products and a sum: 4 * 2^-24 of |a|+|b|
    for y, x, s in ((yq, q, 1), (yk, k, 1), (dq, gq, -1), (dk, gk, -1)):
        want = by_hand(x.detach(), pos, sections, shared, interleaved, sign=s)
        assert (y.double() - want).abs().max() <= 4 * 2 ** -24 * 2 * 6
    one = rot(q, k, pos[:, 0])  # positions for all of a batch
    assert torch.equal(one[0][0], yq[0])


def test_refusals():
    for args in [(8, ()), (8, (0, 2)), (8, (3, 2)), (64, (1,) * 5),
                 (1024, (257,))]:
        with pytest.raises(ValueError):
            AxialRotary(*args)
    with pytest.raises(ValueError):
        AxialRotary(8, (2,), base=0.0)
    rot = AxialRotary(8, (2, 2))
    q, k = torch.zeros(2, 3, 4, 8), torch.zeros(2, 3, 1, 8)
    pos = torch.zeros(2, 2, 3, dtype=torch.int64)
    rot(q, k, pos)
    bad = [(q[0], k, pos), (q, k[:, :2], pos), (q, k[..., :6], pos),
           (q[..., :6], k[..., :6], pos), (q.double(), k.double(), pos),
           (q, k.bfloat16(), pos), (q, k, pos.float()), (q, k, pos[:1]),
           (q, k, pos[:, :1]), (q, k, pos[:, 0, :2])]
    for args in bad:
        with pytest.raises(ValueError):
            rot(*args)


def test_relative_position_only():
    """The product of a rotated query and key depends on their distance."""
    rot = AxialRotary(16, (4, 4))
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(1, 1, 1, 16, generator=g) for _ in range(2))
    dots = []
    for a, b in ((5, 3), (105, 1003)):
        pq = torch.tensor([a + 7, b + 2])[:, None]
        pk = torch.tensor([a, b])[:, None]
        y, _ = rot(q, q, pq)
        z, _ = rot(k, k, pk)
        dots.append((y * z).sum().item())
    assert math.isclose(dots[0], dots[1], abs_tol=1e-4)
