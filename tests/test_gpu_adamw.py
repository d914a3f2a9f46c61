"""fused_adamw kernels vs a 64-bit reference (@gpu)."""

import pytest
import torch

from pytorch_ps_mpi_amd import AdamW, models, ops
from test_adamw import overlapping

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.1)
U = 2.0 ** -24  # half a step of fp32


def _inputs(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda: torch.randn(n, generator=g)  # noqa: E731
    return r() * 0.02, r() * 1e-3, (r() * 1e-3) ** 2, r() * 1e-3


def _reference(p, m, v, g, step, decay, gscale=1.0):
    """64-bit step; with it the sums of magnitudes that bound its rounding."""
    p, m, v, g = (t.double() for t in (p, m, v, g))
    g = g * gscale
    m1, m2 = H["beta1"] * m, (1 - H["beta1"]) * g
    v = H["beta2"] * v + (1 - H["beta2"]) * g * g
    d = v.sqrt() / (1 - H["beta2"] ** step) ** 0.5 + H["eps"]
    f = H["lr"] / (1 - H["beta1"] ** step)
    if decay is not None:
        decay = decay.double().repeat_interleave(256)[:p.numel()]
    else:
        decay = 1.0
    new = p * (1 - H["lr"] * H["wd"] * decay) - f * (m1 + m2) / d
    # roundings: gscale*g, rest, both factors, the sum (m); the same and a
    # square root, division, two factors (update); two of p itself
    mtol = 6 * U * (m1.abs() + m2.abs())
    return (new, m1 + m2, v, mtol, 8 * U * v,
            4 * U * p.abs() + 16 * U * f * (m1.abs() + m2.abs()) / d)


@pytest.mark.parametrize("n", [1, 3, 256, 257, 1000, 100_003, 1 << 20])
@pytest.mark.parametrize("out", [None, torch.bfloat16, torch.float32])
def test_32bit(n, out):
    p, m, v, g = _inputs(n)
    decay = (torch.arange((n + 255) // 256) % 3).float() / 2
    new, rm, rv, mt, vt, pt = _reference(p, m, v, g, 7, decay, 0.5)
    p, m, v, g = (t.to(DEV) for t in (p, m, v, g))
    o = None if out is None else torch.full((n,), 9.0, dtype=out, device=DEV)
    ops.fused_adamw(p, m, v, g, o, step=7, decay=decay.to(DEV), gscale=0.5,
                    **H)
    assert ((p.cpu().double() - new).abs() <= pt).all()
    assert ((m.cpu().double() - rm).abs() <= mt).all()
    assert ((v.cpu().double() - rv).abs() <= vt).all()
    if out is not None:
        assert torch.equal(o, p.to(out))


@pytest.mark.parametrize("n,shift", [(1, 0), (255, 0), (1000, 0), (4096, 1),
                                     (100_003, 0), (1 << 18, 0)])
def test_8bit(n, shift):
    """p from the states' own values; codes are those of the CPU path but for
    values within the fp32 error of a logarithm from their border (3e-5 of the
    distance of two codes: at most a few in 10^5)."""
    p, m, v, g = _inputs(n + shift)
    p, m, v, g = (t[shift:] for t in (p, m, v, g))
    cm, cv = ops.State8.zeros(n, True), ops.State8.zeros(n, False)
    r = ops._mix32(torch.arange(n))
    ops._state8_store(cm, m.contiguous(), r & 0xffff)
    ops._state8_store(cv, v.contiguous(), r >> 16)

    def on_gpu(t):  # with `shift`: no 16-byte alignment
        b = torch.zeros(n + shift, dtype=t.dtype, device=DEV)
        b[shift:] = t.to(DEV)
        return b[shift:]

    gm = ops.State8(on_gpu(cm.codes), cm.scales.to(DEV), True)
    gv = ops.State8(on_gpu(cv.codes), cv.scales.to(DEV), False)
    # 2^(k/8) to one step of fp32, times the maximum
    for a, b in ((gm, cm), (gv, cv)):
        x, y = a.values().cpu(), b.values()
        assert ((x - y).abs() <= 4 * 2 * U * y.abs()).all()
        assert torch.equal(a.values(torch.bfloat16),
                           a.values().to(torch.bfloat16))
    new, rm, rv, mt, vt, pt = _reference(p, gm.values().cpu(),
                                         gv.values().cpu(), g, 7, None)
    gp, gg = on_gpu(p), on_gpu(g)
    go = on_gpu(torch.zeros(n, dtype=torch.bfloat16))
    kw = dict(step=7, seed=11, offset=512, **H)
    ops.fused_adamw(gp, gm, gv, gg, go, **kw)
    assert ((gp.cpu().double() - new).abs() <= pt).all()
    assert torch.equal(go, gp.to(torch.bfloat16))
    cp = p.clone()
    ops.fused_adamw(cp, cm, cv, g.contiguous(), None, **kw)
    for a, b in ((gm, cm), (gv, cv)):
        assert torch.allclose(a.scales.cpu(), b.scales, rtol=8 * 2 * U, atol=0)
        far = (a.codes.cpu().int() - b.codes.int()).abs()
        assert (far != 0).sum().item() <= 2 + 2e-4 * n
        assert far.max().item() <= 1


def test_8bit_parts_equal_whole():
    n = 256 * 40 + 100
    p, m, v, g = (t.to(DEV) for t in _inputs(n))
    got = []
    for cuts in ([0, n], [0, 256, 256 * 17, n]):
        pp, sm, sv = p.clone(), ops.State8.zeros(n, True, DEV), \
            ops.State8.zeros(n, False, DEV)
        for step in (1, 2, 3):
            for a, b in zip(cuts, cuts[1:]):
                ops.fused_adamw(pp[a:b], sm.span(a, b), sv.span(a, b), g[a:b],
                                step=step, offset=a, seed=2, **H)
        got.append((pp, sm.codes, sm.scales, sv.codes, sv.scales))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_8bit_special_values():
    n = 1024
    p = torch.zeros(n, device=DEV)
    g = torch.zeros(n, device=DEV)
    g[0], g[1] = 1e3, 1e-12          # far below the chunk's maximum
    g[300] = 1e-21                   # a second moment below fp32's normal range
    g[512 + 7] = float("inf")
    m, v = ops.State8.zeros(n, True, DEV), ops.State8.zeros(n, False, DEV)
    ops.fused_adamw(p, m, v, g, step=1, **H)
    mv, vv = m.values().cpu(), v.values().cpu()
    assert vv[1] > 0 and vv[2] == 0 and mv[2] == 0
    assert torch.isnan(mv[512:768]).all() and torch.isnan(vv[512:768]).all()
    fine = torch.ones(n, dtype=torch.bool)
    fine[512:768] = False
    assert torch.isfinite(mv[fine]).all() and torch.isfinite(vv[fine]).all()
    assert (p[768:] == 0).all() and torch.isfinite(p[:512]).all()


def test_values_behind_the_end_stay():
    n = 1000
    bufs = [torch.full((n + 24,), 7.0, device=DEV) for _ in range(4)]
    c = [torch.full((n + 24,), 7, dtype=torch.uint8, device=DEV)
         for _ in range(2)]
    sc = [torch.ones(4, device=DEV) for _ in range(2)]
    ops.fused_adamw(bufs[0][:n], ops.State8(c[0][:n], sc[0], True),
                    ops.State8(c[1][:n], sc[1], False), bufs[1][:n],
                    bufs[2][:n], step=1, **H)
    for b in bufs + c:
        assert (b[n:] == 7).all()


def test_graph_replays():
    n = 256 * 30 + 5
    p, _, _, g = (t.to(DEV) for t in _inputs(n))
    eager, cap = [], None
    for captured in (False, True):
        pp, m, v = p.clone(), ops.State8.zeros(n, True, DEV), \
            ops.State8.zeros(n, False, DEV)
        kw = dict(step=3, seed=1, **H)
        if captured:
            ops.fused_adamw(p.clone(), ops.State8.zeros(n, True, DEV),
                            ops.State8.zeros(n, False, DEV), g, **kw)
            torch.cuda.synchronize()
            cap = torch.cuda.CUDAGraph()
            with torch.cuda.graph(cap):
                ops.fused_adamw(pp, m, v, g, **kw)
        for i in range(4):
            if captured:
                cap.replay()
                torch.cuda.synchronize()
                assert torch.equal(pp, eager[i][0])
                assert torch.equal(m.codes, eager[i][1])
                assert torch.equal(v.codes, eager[i][2])
            else:
                ops.fused_adamw(pp, m, v, g, **kw)
                eager.append((pp.clone(), m.codes.clone(), v.codes.clone()))


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_trains_mlp_like_cpu(bits):
    """The optimizer end to end: parameters stay near the CPU path's."""
    got = []
    for dev in ("cpu", DEV):
        torch.manual_seed(0)
        m = models.build_model("mlp", device=dev)
        o = AdamW(m.named_parameters(), lr=1e-3, state_bits=bits,
                  no_decay=lambda n, p: p.dim() < 2)
        x, y = models.synthetic_batch("mlp", 32, device=dev, seed=1)
        for _ in range(3):
            o.zero_grad()
            models.loss_fn("mlp", m, x, y).backward()
            o.step()
        got.append(torch.cat([p.detach().cpu().flatten()
                              for p in m.parameters()]))
    # a step moves a parameter by at most about lr*(1-b1)/sqrt(1-b2) = 3.2 lr;
    # where a gradient is within rounding of zero its sign is not determined
    assert (got[0] - got[1]).abs().max() <= 2 * 3 * 3.2e-3
    assert (got[0] - got[1]).norm() <= 1e-2 * got[0].norm()


def test_shared_memory_is_refused():
    overlapping(DEV)
