"""fused_gated_residual kernels against 64 bits (@gpu).

Bounds.  e is half a step of the type, S = 64 * 2^-24 covers fp32 arithmetic
(sums over lanes, waves and blocks: some 30 roundings); `_bounds` carries the
error of the normed values through the backward pass term by term.
"""

import pytest
import torch

from pytorch_ps_mpi_amd.ops.ln import _join_plain
from test_join import call, inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
S = 64 * 2.0 ** -24
NAMES = ("x", "u", "w", "b", "gate", "pw", "pb")


def _reference(t, scale, kind, eps=1e-5):
    """64-bit results by autograd, and a bound for each."""
    d = {n: None if v is None else v.double() for n, v in t.items()}
    leaves = {n: d[n].requires_grad_() for n in NAMES if d[n] is not None}
    y, h = _join_plain(d["x"], d["u"], d["w"], d["b"], d["gate"], d["pw"],
                       d["pb"], scale, eps, kind)
    grads = torch.autograd.grad((y, h), list(leaves.values()),
                                (d["gy"], d["gh"]))
    want = {"y": y.detach(), "h": h.detach(),
            **{"d" + n: v for n, v in zip(leaves, grads)}}
    return want, _bounds({n: None if v is None else v.detach()
                          for n, v in d.items()}, want, t["x"].dtype, scale,
                         kind, eps)


def _stats(f, kind, eps):
    mu = f.mean(-1, keepdim=True) if kind == "layer" else 0.0
    r = ((f - mu) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    return (f - mu) * r, r


def _bounds(d, want, dtype, scale, kind, eps):
    e = torch.finfo(dtype).eps / 2
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    n = d["u"]
    if d["pw"] is not None:
        uh, ur = _stats(d["u"], kind, eps)
        n = uh * d["pw"] + (0 if d["pb"] is None else d["pb"])
    y = want["y"]
    gate = torch.ones_like(y) if d["gate"] is None else d["gate"]
    hat, r = _stats(y, kind, eps)
    mag = scale * d["x"].abs() + (gate * n).abs()
    top = mag.amax(-1, keepdim=True)  # statistics see every element
    tol = {"y": e * y.abs() + S * (mag + gate.abs()),
           "h": e * want["h"].abs() + S * (
               (mag + top) * r * d["w"].abs() + want["h"].abs() + 1)}
    off = S * ((mag + top) * r + hat.abs())       # of the normed value
    k = (d["gh"] * d["w"])
    c2 = mean(k * hat).abs()
    et = r * (off * c2 + hat.abs() * mean(k.abs() * off)
              + S * (k.abs() + mean(k.abs()) + hat.abs() * mean(
                  (k * hat).abs()))) + S * d["gy"].abs()
    t = (want["dx"] / scale).abs()
    tol["dx"] = e * want["dx"].abs() + scale * et + S * t
    rows = (0, 1)
    tol["dw"] = e * want["dw"].abs() + (d["gh"].abs() * off).sum(rows) \
        + S * (d["gh"] * hat).abs().sum(rows)
    if d["b"] is not None:
        tol["db"] = e * want["db"].abs() + S * d["gh"].abs().sum(rows)
    eg = et * n.abs() + S * t * (n.abs() + 1)
    if d["gate"] is not None:
        g = want["dgate"]
        if g.shape == y.shape:
            s = eg
        elif g.dim() == 1:
            s = eg.sum(rows)
        else:
            s = eg.sum(1, keepdim=True)
        tol["dgate"] = e * g.abs() + s
    en = et * gate.abs() + S * t * gate.abs()
    tn = t * gate.abs()
    if d["pw"] is not None:
        tol["dpw"] = e * want["dpw"].abs() + (en * uh.abs()).sum(rows) \
            + S * (tn * (uh.abs() + 1)).sum(rows)
        if d["pb"] is not None:
            tol["dpb"] = e * want["dpb"].abs() + (en + S * tn).sum(rows)
        en, tn = en * d["pw"].abs(), tn * d["pw"].abs()
        en = ur * (en + mean(en) + uh.abs() * mean(en * uh.abs())
                   + S * (tn + mean(tn) + (uh.abs() + 1) * mean(
                       tn * (uh.abs() + 1))))
    tol["du"] = e * want["du"].abs() + en
    return tol


def _run(t, scale, kind):
    dev = {n: None if v is None else v.to(DEV).requires_grad_(n in NAMES)
           for n, v in t.items()}
    y, h = call(dev, scale, kind)
    leaves = {n: dev[n] for n in NAMES if dev[n] is not None}
    grads = torch.autograd.grad((y, h), list(leaves.values()),
                                (dev["gy"], dev["gh"]))
    return {"y": y.detach(), "h": h.detach(),
            **{"d" + n: v for n, v in zip(leaves, grads)}}


def _check(t, scale, kind):
    want, tol = _reference(t, scale, kind)
    got = _run(t, scale, kind)
    for n in want:
        assert got[n].shape == want[n].shape, n
        err = (got[n].cpu().double() - want[n]).abs()
        assert (err <= tol[n]).all(), (n, err.max(), (err / tol[n]).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "token"])
@pytest.mark.parametrize("post", [False, True])
def test_every_form(dtype, kind, gate, post):
    _check(inputs(3, 17, 768, dtype, gate, post, kind == "layer"), 0.7, kind)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,D", [
    (1, 1, 1), (1, 1, 8), (2, 3, 5), (1, 9, 100), (4, 197, 64), (2, 50, 512),
    (1, 70, 513), (2, 33, 1000), (1, 40, 1024), (1, 21, 1032), (2, 9, 2048),
    (1, 11, 2500), (1, 6, 4096), (2, 3, 4104), (1, 5, 8191), (1, 7, 8192),
    (700, 2, 64), (1, 3000, 72),
])
@pytest.mark.parametrize("gate", ["channel", "sample"])
def test_sizes(dtype, B, T, D, gate):
    # one element: nothing is left after the mean; take the rms kind there
    kind = "rms" if D == 1 else "layer"
    _check(inputs(B, T, D, dtype, gate, True, True, seed=D), 1.0, kind)


def test_far_mean_keeps_its_variance():
    """A large common offset: the variance is taken about the mean."""
    t = inputs(2, 8, 256, torch.float32, "none", False, True)
    t["x"] = t["x"] + 1000.0
    _check(t, 1.0, "layer")


@pytest.mark.parametrize("which", ["gy", "gh"])
def test_one_gradient_only(which):
    t = inputs(2, 9, 96, torch.float32, "channel", True, True)
    full = dict(t)
    full["gy" if which == "gh" else "gh"] = torch.zeros_like(t["gy"])
    want, tol = _reference(full, 0.7, "layer")
    dev = {n: None if v is None else v.to(DEV).requires_grad_(n in NAMES)
           for n, v in t.items()}
    y, h = call(dev, 0.7)
    out, g = (y, dev["gy"]) if which == "gy" else (h, dev["gh"])
    leaves = [n for n in NAMES if dev[n] is not None]
    grads = torch.autograd.grad(out, [dev[n] for n in leaves], g,
                                allow_unused=True)
    for n, v in zip(leaves, grads):
        if v is None:
            assert which == "gy" and n in ("w", "b")
            assert want["d" + n].abs().max() == 0
        else:
            err = (v.cpu().double() - want["d" + n]).abs()
            assert (err <= tol["d" + n]).all(), n


def test_partial_needs_and_views():
    t = inputs(2, 9, 96, torch.bfloat16, "sample", True, True)
    want = _run(t, 0.7, "layer")
    dev = {n: None if v is None else v.to(DEV) for n, v in t.items()}
    dev["u"].requires_grad_()
    dev["pw"].requires_grad_()
    # a transposed x, a sliced weight, an expanded gradient
    dev["x"] = dev["x"].transpose(0, 1).contiguous().transpose(0, 1)
    dev["w"] = torch.stack([dev["w"], dev["w"]], 1)[:, 0]
    y, h = call(dev, 0.7)
    du, dpw = torch.autograd.grad((y, h), (dev["u"], dev["pw"]),
                                  (dev["gy"], dev["gh"]))
    assert torch.equal(y, want["y"]) and torch.equal(h, want["h"])
    assert torch.equal(du, want["du"]) and torch.equal(dpw, want["dpw"])


def test_repeats_bit_for_bit_and_in_graphs():
    t = inputs(4, 300, 768, torch.bfloat16, "channel", True, True)
    a, b = _run(t, 0.7, "layer"), _run(t, 0.7, "layer")
    for n in a:
        assert torch.equal(a[n], b[n]), n
    dev = {n: v.to(DEV).requires_grad_(n in NAMES) for n, v in t.items()}
    leaves = [dev[n] for n in NAMES]

    def step():
        y, h = call(dev, 0.7)
        g = torch.autograd.grad((y, h), leaves, (dev["gy"], dev["gh"]))
        return (y.detach(), h.detach(), *g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            dev["u"].mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        for p, q in zip(got, step()):
            assert torch.equal(p, q)


def test_empty_and_refusals():
    x = torch.zeros(0, 4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    y, h = call(dict(x=x, u=x, w=w, b=None, gate=torch.zeros(0, 1, 8,
                     device=DEV), pw=None, pb=None))
    assert y.shape == h.shape == x.shape
    ok = inputs(1, 2, 8, torch.float32, "none", False, False)
    dev = {n: None if v is None else v.to(DEV) for n, v in ok.items()}
    for bad in (dict(w=dev["w"].cpu()),
                {n: v.double() for n, v in dev.items() if v is not None},
                {n: v.half() for n, v in dev.items() if v is not None}):
        with pytest.raises(ValueError):
            call({**dev, **bad})
    big = inputs(1, 1, 8200, torch.float32, "none", False, False)
    with pytest.raises(ValueError):
        call({n: None if v is None else v.to(DEV) for n, v in big.items()})


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "token"])
def test_longest_rows_over_several_rows_a_block(dtype, gate):
    """Rows past 4096 with both norms keep their sums in LDS; 256 blocks take
    these rows, three or two each."""
    B, T = (2, 300) if gate == "sample" else (1, 600)
    _check(inputs(B, T, 5000, dtype, gate, True, True), 0.9, "layer")
