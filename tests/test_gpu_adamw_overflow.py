"""8-bit AdamW states whose second moment alone leaves fp32's range (@gpu)."""

import pytest
import torch

from pytorch_ps_mpi_amd import ops

pytestmark = pytest.mark.gpu


def test_one_state_overflows():
    """A gradient of 1e21 squares to an infinity: the second moment of its 256
    elements reads as NaN, the first one goes on, on both paths; one step
    later both parameters are NaN there and nowhere else."""
    n = 700
    g = torch.randn(n, generator=torch.Generator().manual_seed(0))
    g[300], g[310] = 1e21, 0.0
    got = []
    for dev in ("cpu", "cuda:0"):
        p = torch.zeros(n, device=dev)
        m, v = ops.State8.zeros(n, True, dev), ops.State8.zeros(n, False, dev)
        first = None
        for step in (1, 2):
            ops.fused_adamw(p, m, v, g.to(dev), lr=1e-3, step=step)
            first = first or (p.isfinite().cpu(), m.values().isfinite().cpu(),
                              v.values().isfinite().cpu())
        got.append((*first, p.isfinite().cpu(), m.values().isfinite().cpu(),
                    v.values().isfinite().cpu()))
        assert torch.allclose(m.values().cpu()[300], g[300] * 0.19, rtol=0.2)
    fine = torch.ones(n, dtype=torch.bool)
    fine[256:512] = False
    every = torch.ones(n, dtype=torch.bool)
    for p1, m1, v1, p2, m2, v2 in got:
        assert torch.equal(p1, every) and torch.equal(m1, every)
        assert torch.equal(v1, fine) and torch.equal(p2, fine)
        assert torch.equal(m2, every) and torch.equal(v2, fine)
