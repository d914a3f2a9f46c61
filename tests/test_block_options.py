"""The models' options that use windowed attention, rotary axes and gated
residual norms, trained by AdamW: CPU runs, and GPU against CPU."""

import pytest
import torch

from pytorch_ps_mpi_amd import AdamW, models
from pytorch_ps_mpi_amd.models.gpt2 import GPT2
from pytorch_ps_mpi_amd.models.vit import ViT

GPT = dict(vocab=101, ctx=96, dim=256, depth=2, heads=4, window=24, sinks=2,
           kv_heads=2, rotary=True, layer_scale=0.5)
VIT = dict(img=48, patch=16, dim=128, depth=2, heads=2, num_classes=7,
           rotary=True, layer_scale=0.5)


def _gpt(**kw):
    torch.manual_seed(0)
    return GPT2(**{**GPT, **kw})


def _vit(**kw):
    torch.manual_seed(0)
    return ViT(**{**VIT, **kw})


def _data(kind, device="cpu"):
    g = torch.Generator().manual_seed(1)
    if kind == "gpt":
        t = torch.randint(0, 101, (3, 78), generator=g)
        return t[:, :-1].to(device), t[:, 1:].to(device)
    return (torch.randn(4, 3, 48, 48, generator=g).to(device),
            torch.randint(0, 7, (4,), generator=g).to(device))


def _loss(kind, m, x, y):
    if kind == "gpt":
        return m.loss(x, y)
    return torch.nn.functional.cross_entropy(
        m(x.to(m.head.weight.dtype)).float(), y)


def test_wide_window_is_the_full_model():
    """A window that covers the context, one key head a query head: the same
    function as the full causal path; a gate of one changes nothing."""
    torch.manual_seed(0)
    a = GPT2(vocab=64, ctx=32, dim=64, depth=2, heads=2)
    b = GPT2(vocab=64, ctx=32, dim=64, depth=2, heads=2, window=32,
             layer_scale=1.0)
    b.load_state_dict({**b.state_dict(), **a.state_dict()})
    x = torch.randint(0, 64, (2, 20))
    assert torch.allclose(a(x), b(x), atol=1e-5)


def test_window_limits_what_a_token_sees():
    """Two layers of window 4 reach 6 tokens back; with a first token that
    stays visible a change of it reaches everything."""
    for sinks, reaches in ((0, False), (1, True)):
        m = _gpt(window=4, sinks=sinks).eval()
        x = torch.randint(0, 101, (1, 30), generator=torch.Generator()
                          .manual_seed(2))
        z = x.clone()
        z[0, 0] = (z[0, 0] + 1) % 101
        d = (m(x) - m(z)).abs().amax(2)[0]
        assert (d[7:] > 0).all() if reaches else (d[7:] == 0).all()


@pytest.mark.parametrize("bad", [dict(kv_heads=3), dict(kv_heads=0),
                                 dict(window=0), dict(sinks=-1)])
def test_refusals(bad):
    with pytest.raises(ValueError):
        _gpt(**bad)


def test_block_alone_takes_positions_by_itself():
    m = _gpt(layer_scale=None)
    x = torch.randn(2, 9, 256)
    pos = torch.arange(9)[None]
    assert torch.equal(m.blocks[0](x), m.blocks[0](x, pos))


def test_registry_passes_options():
    m = models.build_model("vit_b16", num_classes=10, rotary=True,
                           layer_scale=0.1)
    assert m.blocks[0].rotary is not None and \
        m.blocks[3].g1[0].item() == pytest.approx(0.1)


@pytest.mark.parametrize("kind", ["gpt", "vit"])
@pytest.mark.parametrize("bits", [8, 32])
def test_trains_on_cpu(kind, bits):
    m = _gpt() if kind == "gpt" else _vit()
    o = AdamW(m.named_parameters(), lr=1e-3, state_bits=bits,
              no_decay=lambda n, p: p.dim() < 2)
    x, y = _data(kind)
    before = [p.detach().clone() for p in m.parameters()]
    for _ in range(2):
        o.zero_grad()
        loss = _loss(kind, m, x, y)
        loss.backward()
        o.step()
    assert torch.isfinite(loss)
    for a, p in zip(before, m.parameters()):
        assert torch.isfinite(p).all() and not torch.equal(a, p)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gpt", "vit"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_gradients_are_the_cpus(kind, dtype):
    """Loss and every gradient against the fp32 CPU path on the same weights.
    In bf16 a value passes some 40 roundings of at most 2^-8 forward and as
    many backward; independent ones add to 2^-8 sqrt(80) = 3.5%, of which a
    small gradient behind cancelling sums sees a multiple: 4 times that."""
    m = _gpt() if kind == "gpt" else _vit()
    m = m.to(dtype)  # the same rounded weights on both sides
    c = _gpt() if kind == "gpt" else _vit()
    c.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    _loss(kind, c, *_data(kind)).backward()
    g = m.to("cuda:0")
    _loss(kind, g, *_data(kind, "cuda:0")).backward()
    # fp32: sums of up to 10^4 products, 2^-24 sqrt(10^4), through 40 steps
    tol = 1e-3 if dtype == torch.float32 else 4 * 0.035
    for (n, a), b in zip(c.named_parameters(), g.parameters()):
        d = (b.grad.cpu().float() - a.grad).norm()
        assert d <= tol * a.grad.norm() + 1e-7, (n, d / a.grad.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gpt", "vit"])
@pytest.mark.parametrize("bits", [8, 32])
def test_gpu_trains(kind, bits):
    """The operators together under the optimizer."""
    m = (_gpt() if kind == "gpt" else _vit()).to("cuda:0", torch.bfloat16)
    o = AdamW(m.named_parameters(), lr=1e-3, state_bits=bits, seed=3,
              no_decay=lambda n, p: p.dim() < 2)
    x, y = _data(kind, "cuda:0")
    before = o.flat.master.clone()
    for _ in range(3):
        o.zero_grad()
        loss = _loss(kind, m, x, y)
        loss.backward()
        o.step()
    assert torch.isfinite(loss) and torch.isfinite(o.flat.master).all()
    moved = (o.flat.master - before).abs()
    # a step is at most lr (1-b1)/sqrt(1-b2) = 3.2 lr, and decay
    assert 0 < moved.max() <= 3 * (3.2e-3 + 1e-5 * before.abs().max()) * 1.01
    for name, p, off, n in o.flat.entries:
        assert torch.equal(p.detach().flatten(),
                           o.flat.master[off:off + n].bfloat16())
