"""fused_gated_residual: the CPU path (the oracle) and its refusals."""

import pytest
import torch

from pytorch_ps_mpi_amd.ops.ln import FusedLayerNorm, fused_gated_residual


def inputs(B, T, D, dtype, gate, post, bias, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = dict(x=r(B, T, D) + 0.3, u=r(B, T, D) * 0.5 - 0.1, w=1 + 0.1 * r(D),
             b=0.1 * r(D) if bias else None, gate=None,
             pw=1 + 0.1 * r(D) if post else None,
             pb=0.1 * r(D) if post and bias else None)
    shape = dict(none=None, channel=(D,), sample=(B, 1, D),
                 token=(B, T, D))[gate]
    if shape:
        t["gate"] = 0.5 + 0.3 * r(*shape)
    t["gy"], t["gh"] = 0.1 * r(B, T, D), 0.1 * r(B, T, D)
    return {n: None if v is None else v.to(dtype) for n, v in t.items()}


def call(t, scale=0.7, kind="layer"):
    return fused_gated_residual(t["x"], t["u"], t["w"], t["b"],
                                gate=t["gate"], post_weight=t["pw"],
                                post_bias=t["pb"], scale=scale, kind=kind)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "token"])
@pytest.mark.parametrize("post", [False, True])
def test_gradients_against_differences(kind, gate, post):
    t = inputs(2, 3, 5, torch.float64, gate, post, True)
    names = [n for n in ("x", "u", "w", "b", "gate", "pw", "pb")
             if t[n] is not None]

    def f(*v):
        return call({**t, **dict(zip(names, v))}, kind=kind)

    assert torch.autograd.gradcheck(
        f, [t[n].requires_grad_() for n in names])


def test_is_the_blocks_own_formula():
    """LayerNorm after a residual sum, as the models write it."""
    t = inputs(2, 4, 32, torch.float32, "none", False, True)
    ln = FusedLayerNorm(32)
    with torch.no_grad():
        ln.weight.copy_(t["w"])
        ln.bias.copy_(t["b"])
    y, h = call(t, scale=1.0)
    assert torch.equal(y, t["x"] + t["u"])
    assert torch.allclose(h, ln(t["x"] + t["u"]), atol=1e-6)


def test_refusals():
    t = inputs(2, 3, 8, torch.float32, "none", False, False)
    x, u, w = t["x"], t["u"], t["w"]
    fused_gated_residual(x, u, w)
    bad = [
        ((x, u[:1], w), {}), ((x, u, w[:4]), {}), ((x, u, w, w[:4]), {}),
        ((x, u.bfloat16(), w), {}), ((x, u, w.bfloat16()), {}),
        ((x, u, w), dict(kind="batch")), ((x, u, w), dict(post_bias=w)),
        ((x, u, w), dict(gate=w[:4])), ((x, u, w), dict(gate=x[:, :1, :4])),
        ((x, u, w), dict(gate=x[:1])), ((x, u, w), dict(gate=w.double())),
        ((x[..., :0], u[..., :0], w[:0]), {}),
        ((x[0], u[0], w), dict(gate=x[:, :1])),
    ]
    for args, kw in bad:
        with pytest.raises(ValueError):
            fused_gated_residual(*args, **kw)
