"""Blocks with gates on their branches (layer_scale), alone and in a model."""

import pytest
import torch

from pytorch_ps_mpi_amd.models.gpt2 import GPT2, CausalBlock
from pytorch_ps_mpi_amd.models.vit import Block, ViT


def _block(cls):
    torch.manual_seed(0)
    b = cls(64, 2, layer_scale=0.5)
    with torch.no_grad():  # gates that differ by channel and branch
        b.g1.copy_(torch.linspace(-1, 1, 64))
        b.g2.copy_(torch.linspace(2, 0.1, 64))
    return b


@pytest.mark.parametrize("cls", [CausalBlock, Block])
def test_block_alone_has_its_gates(cls):
    """As in a model: x + g1 * attention, then + g2 * mlp."""
    b = _block(cls)
    x = torch.randn(2, 9, 64, requires_grad=True)
    y = x + b.g1 * b.attend(b.n1(x))
    want = y + b.g2 * b.mlp(b.n2(y))
    got = b(x)
    # values of up to 10, sums of 256 products: 10 * sqrt(256) * 2^-24 = 1e-5
    assert torch.allclose(got, want, atol=1e-5)
    leaves = [x, *b.parameters()]
    go = torch.randn_like(got)
    for a, c in zip(torch.autograd.grad(got, leaves, go),
                    torch.autograd.grad(want, leaves, go)):
        # as much again in each of some ten steps back
        assert torch.allclose(a, c, atol=1e-4)
    with torch.no_grad():
        b.g1.zero_()
        b.g2.zero_()
    assert torch.equal(b(x), x)
    h = torch.nn.LayerNorm(64)
    s, n = b.joined(x, b.n1(x), h)
    assert torch.equal(s, x) and torch.allclose(n, h(x), atol=1e-5)


def _models():
    torch.manual_seed(0)
    yield (GPT2(vocab=31, ctx=16, dim=64, depth=3, heads=2, layer_scale=0.5),
           torch.randint(0, 31, (2, 9)))
    yield (ViT(img=16, patch=8, dim=64, depth=3, heads=2, num_classes=5,
               layer_scale=0.5), torch.randn(2, 3, 16, 16))


def test_models_call_their_gated_blocks():
    """Hooks of a block and wrappers of its forward see every step, and what
    they return counts."""
    for m, x in _models():
        want, seen = m(x), []
        for i, b in enumerate(m.blocks):
            b.register_forward_hook(
                lambda mod, args, out, i=i: seen.append((i, len(out))))
        assert torch.equal(m(x), want)
        assert seen == [(0, 2), (1, 2), (2, 2)]
        inner = m.blocks[1].forward
        m.blocks[1].forward = lambda *a, **k: torch.utils.checkpoint \
            .checkpoint(inner, *a, use_reentrant=False, **k)
        got = m(x)
        assert torch.equal(got, want)
        got.sum().backward()
        assert all(torch.isfinite(p.grad).all() for p in m.parameters())
        m.blocks[2].register_forward_hook(
            lambda mod, args, out: (out[0], out[1] * 0))
        assert torch.equal(m(x)[0], m(x)[1])


@pytest.mark.parametrize("alone", [False, True])
def test_gated_blocks_under_autocast(alone):
    """Branches come back in bf16, the residual stream stays in fp32, as
    without gates: a model with gates of one is the default one.  Both paths
    round the same values to bf16; where they lie within fp32 rounding of a
    border they differ by a step, 2^-7, of one value of many: the norm of the
    difference stays under that of all."""
    for make, x in (
            (lambda **k: GPT2(vocab=31, ctx=16, dim=64, depth=2, heads=2, **k),
             torch.randint(0, 31, (2, 9))),
            (lambda **k: ViT(img=16, patch=8, dim=64, depth=2, heads=2,
                             num_classes=5, **k),
             torch.randn(2, 3, 16, 16))):
        torch.manual_seed(0)
        a, b = make(), make(layer_scale=1.0)
        b.load_state_dict({**b.state_dict(), **a.state_dict()})
        if alone:
            a, b = a.blocks[1], b.blocks[1]
            x = torch.randn(2, 7, 64)
        got = []
        for m in (a, b):
            with torch.autocast("cpu", dtype=torch.bfloat16):
                y = m(x)
            y.float().square().sum().backward()
            got.append((y.detach().float(), dict(m.named_parameters())))
        assert (got[0][0] - got[1][0]).norm() <= 2 ** -7 * got[0][0].norm()
        for n, p in got[0][1].items():
            g = got[1][1][n].grad
            assert (p.grad - g).norm() <= 2 ** -5 * p.grad.norm() + 1e-6, n
