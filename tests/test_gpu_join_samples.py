"""fused_gated_residual with a gate for each of very many samples (@gpu)."""

import pytest
import torch

from test_gpu_join import DEV, _reference, _run
from test_join import call, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [65531, 140_000])
@pytest.mark.parametrize("dtype,post", [(torch.bfloat16, False),
                                        (torch.float32, True)])
def test_more_samples_than_a_grid_has_rows(B, dtype, post):
    """One sum for each sample's gate: more than 65535 of them take several
    launches.  Whole-batch sums pass B / 32 parts one after another, in place
    of the 64 roundings that test_gpu_join counts; their bound grows by
    that."""
    t = inputs(B, 2, 8, dtype, "sample", post, True)
    want, tol = _reference({n: None if v is None else v.to(DEV)
                            for n, v in t.items()}, 0.7, "layer")
    got = _run(t, 0.7, "layer")
    for n in want:
        far = B / 32 / 64 if n in ("dw", "db", "dpw", "dpb") else 0
        err = (got[n].double() - want[n]).abs()
        assert (err <= tol[n] * (1 + far)).all(), (n, err.max())


def test_sums_of_wide_rows_for_many_samples():
    """20000 gates of 8192 would be 5 * 2^30 threads.  The last samples by
    themselves give the same dx and du.  A gate's sum has two products
    t * u, t = dx / scale: one block adds the second one by a fused operation,
    two blocks leave it to the sum of parts, rounded first.  So the sums are
    off by 2 * 2^-24 of their magnitudes (twice that covers dx's own rounding),
    which may carry one over the border of a bf16 step, 2^-7 of the value."""
    B, D = 20_000, 8192
    g = torch.Generator(device=DEV).manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV,  # noqa: E731
                                dtype=torch.bfloat16)
    x, u, gy, gh = (mk(B, 2, D) for _ in range(4))
    w, gate = mk(D), mk(B, 1, D)

    def grads(part):
        t = [v[part].clone().requires_grad_() for v in (x, u, gate)]
        y, h = call(dict(x=t[0], u=t[1], w=w, b=None, gate=t[2], pw=None,
                         pb=None))
        return torch.autograd.grad((y, h), t, (gy[part], gh[part]))

    got = grads(slice(None))
    for part in (slice(0, 5), slice(8190, 8195), slice(B - 5, B)):
        (dx, du, dg), want = (a[part] for a in got), grads(part)
        assert torch.equal(dx, want[0]) and torch.equal(du, want[1])
        mag = (dx.double() / 0.7 * u[part].double()).abs().sum(1, True)
        err = (dg.double() - want[2].double()).abs()
        assert (err <= 2.0 ** -7 * want[2].double().abs()
                + 2.0 ** -22 * mag).all()
