"""AdamW over the packed flat space (CPU path): torch.optim.AdamW's formula,
8-bit states, checkpoints, bucketing, refusals."""

import math

import pytest
import torch

from pytorch_ps_mpi_amd import MPI_PS, AdamW, models, ops
from pytorch_ps_mpi_amd.utils import checkpoint

STEP = 2 ** 0.125  # ratio of neighbouring codes


def _train(model, opt, steps=4, seed=1, batch=16):
    x, y = models.synthetic_batch("mlp", batch, seed=seed)
    for _ in range(steps):
        opt.zero_grad()
        models.loss_fn("mlp", model, x, y).backward()
        opt.step()


def _flat(m):
    return torch.cat([p.detach().flatten() for p in m.parameters()])


def test_parity_with_torch():
    torch.manual_seed(0)
    m1 = models.build_model("mlp")
    torch.manual_seed(0)
    m2 = models.build_model("mlp")
    o1 = AdamW(m1.named_parameters(), lr=1e-3, weight_decay=0.1,
               no_decay=lambda n, p: p.dim() < 2)
    o2 = torch.optim.AdamW(
        [dict(params=[p for p in m2.parameters() if p.dim() > 1],
              weight_decay=0.1),
         dict(params=[p for p in m2.parameters() if p.dim() < 2],
              weight_decay=0.0)], lr=1e-3)
    _train(m1, o1)
    _train(m2, o2)
    assert torch.allclose(_flat(m1), _flat(m2), atol=1e-6)


def test_factory():
    m = models.build_model("mlp")
    o = MPI_PS(m.named_parameters(), optim="adamw", state_bits=8)
    assert isinstance(o, AdamW) and o.state_bits == 8


def test_8bit_states_are_neighbours_and_unbiased():
    """Each stored value is one of the two codes around the real one, and the
    mean relative error is that of a fair choice between them."""
    torch.manual_seed(0)
    n = 1 << 18
    for signed in (True, False):
        st = ops.State8.zeros(n, signed)
        x = torch.rand(n) * 0.9 + 0.1      # within range of the lowest code
        if signed:
            x = x * torch.where(torch.rand(n) < 0.5, -1.0, 1.0)
        r = ops._mix32(torch.arange(n))
        ops._state8_store(st, x, r & 0xffff)
        y = st.values()
        ratio = (y / x).double()
        # neighbours are a factor 2^(1/8) apart; 1e-4 covers fp32 logarithms
        assert ratio.min() > 1 / STEP - 1e-4 and ratio.max() < STEP + 1e-4
        # one error has a deviation of at most (STEP-1)/2: six deviations
        assert abs(ratio.mean().item() - 1) < 6 * (STEP - 1) / 2 / math.sqrt(n)


def test_8bit_average_is_not_frozen():
    """A second moment decays at its rate though a step (0.1%) is far below
    the distance of two codes (9%)."""
    n, steps = 1 << 14, 300
    m, v = ops.State8.zeros(n, True), ops.State8.zeros(n, False)
    p = torch.zeros(n)
    g = torch.full((n,), 0.5)
    g[::256] = 1.0  # the maxima, which the others are measured by
    ops.fused_adamw(p, m, v, g, lr=0.0, beta2=0.5, step=1, wd=0.0)
    v0 = v.values().double().mean()
    for t in range(2, steps + 2):
        ops.fused_adamw(p, m, v, torch.zeros(n), lr=0.0, beta2=0.999, step=t,
                        wd=0.0)
    # per element the spread is sqrt(steps * 0.001 * 0.09) ~ 16%; the mean
    # over 2^14 of them is within 0.8% at six deviations
    assert abs(v.values().double().mean() / v0 / 0.999 ** steps - 1) < 0.008


def test_8bit_special_values():
    n = 512
    st = ops.State8.zeros(n, False)
    x = torch.zeros(n)
    x[0], x[1], x[300] = 1.0, 1e-30, 1e-42
    ops._state8_store(st, x, torch.zeros(n, dtype=torch.int64))
    y = st.values()
    assert y[1] > 0 and y[2] == 0          # not zero stays not zero
    assert y[300] == x[300] and (y[256:] > 0).sum() == 1
    x[5] = float("inf")
    ops._state8_store(st, x, torch.zeros(n, dtype=torch.int64))
    y = st.values()
    assert torch.isnan(y[:256]).all() and torch.isfinite(y[256:]).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_bucketing_does_not_change_results(bits):
    got = []
    threads = torch.get_num_threads()
    torch.set_num_threads(1)  # several split the elementwise loops anew
    for mb in (50, 0.0001):
        torch.manual_seed(0)
        m = models.build_model("mlp")
        o = AdamW(m.named_parameters(), lr=1e-3, state_bits=bits,
                  bucket_mb=mb, seed=3, no_decay=lambda n, p: p.dim() < 2)
        _train(m, o, steps=3)
        got.append((len(o.flat.buckets), _flat(m),
                    [t.clone() for t in o._state_tensors().values()]))
    torch.set_num_threads(threads)
    assert got[0][0] != got[1][0]
    assert torch.equal(got[0][1], got[1][1])
    for a, b in zip(got[0][2], got[1][2]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_resume(tmp_path, bits):
    torch.manual_seed(0)
    m1 = models.build_model("mlp")
    o1 = AdamW(m1.named_parameters(), lr=1e-3, state_bits=bits, seed=5)
    _train(m1, o1, steps=3)
    path = str(tmp_path / "ck.pt")
    checkpoint.save(path, o1)
    torch.manual_seed(9)
    m2 = models.build_model("mlp")
    o2 = AdamW(m2.named_parameters(), lr=1e-3, state_bits=bits)
    checkpoint.load(path, o2)
    _train(m1, o1, steps=2, seed=4)
    _train(m2, o2, steps=2, seed=4)
    assert torch.equal(_flat(m1), _flat(m2))
    m3 = models.build_model("mlp")
    o3 = AdamW(m3.named_parameters(), state_bits=40 - bits)
    before = _flat(m3)
    with pytest.raises(ValueError, match="bit AdamW states"):
        checkpoint.load(path, o3)
    assert torch.equal(_flat(m3), before)


def overlapping(dev):
    """Calls of fused_adamw in which a written tensor shares memory."""
    n = 512
    t = lambda k=n: torch.zeros(k, device=dev)  # noqa: E731
    a, b, c = t(), t(), t(3 * n)
    e8, f8 = (ops.State8.zeros(n, s, dev) for s in (True, False))
    bad = [
        ((a, b, b, t()), {}), ((a, a, b, t()), {}), ((a, b, t(), a), {}),
        ((a, b, t(), b), {}), ((a, b, t(), t()), dict(p_out=a)),
        ((c[:n], c[256:256 + n], t(), t()), {}),
        ((a, e8, ops.State8(e8.codes, t(2), False), t()), {}),
        ((a, e8, ops.State8(f8.codes, e8.scales, False), t()), {}),
        ((a, b, t(), t()), dict(decay=b[:2])),
    ]
    for args, kw in bad:
        with pytest.raises(ValueError, match="share memory"):
            ops.fused_adamw(*args, lr=1e-3, **kw)
    # neighbours, and a gradient that holds the factors: fine
    ops.fused_adamw(c[:n], c[n:2 * n], c[2 * n:], a, decay=a[:2], lr=1e-3)


def test_shared_memory_is_refused():
    overlapping("cpu")


def test_refusals():
    n = 512
    t = lambda k=n: torch.zeros(k)  # noqa: E731
    s8 = ops.State8.zeros
    ok = dict(lr=1e-3)
    ops.fused_adamw(t(), t(), t(), t(), None, **ok)
    ops.fused_adamw(t(0), t(0), t(0), t(0), None, **ok)
    bad = [
        ((t(), t(), s8(n, False), t()), {}),
        ((t(), s8(n, False), s8(n, True), t()), {}),
        ((t(), s8(256, True), s8(256, False), t()), {}),
        ((t(), t(256), t(), t()), {}),
        ((t(), t(), t(), t().bfloat16()), {}),
        ((t(1024)[::2], t(), t(), t()), {}),
        ((t(), t(), t(), t()), dict(step=0)),
        ((t(), t(), t(), t()), dict(beta2=1.0)),
        ((t(), t(), t(), t()), dict(decay=t(1))),
        ((t(), t(), t(), t()), dict(p_out=t(8))),
        ((t(), t(), t(), t()), dict(p_out=t().half())),
        ((t(), s8(n, True), s8(n, False), t()), dict(offset=100)),
        ((t(), t(), t(), t()), dict(offset=-256)),
    ]
    for args, kw in bad:
        with pytest.raises(ValueError):
            ops.fused_adamw(*args, **ok, **kw)
    for codes, scales in [(t(), t(2)), (t().byte(), t(3)),
                          (t().byte(), t(2).double()),
                          (t(1024).byte()[::2], t(2))]:
        with pytest.raises(ValueError):
            ops.State8(codes, scales, True)
    with pytest.raises(ValueError):
        s8(n, True).span(100, 512)
    with pytest.raises(ValueError):
        s8(n, True).span(0, 100)
    with pytest.raises(ValueError):
        s8(n, True).values(torch.float16)
    with pytest.raises(ValueError):
        AdamW(models.build_model("mlp").named_parameters(), state_bits=4)


def _worker(rank, port, mode, bits, out):
    import os
    os.environ.update(RANK=str(rank), WORLD_SIZE="2", LOCAL_RANK=str(rank),
                      MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    import torch.distributed as dist
    from pytorch_ps_mpi_amd import init_distributed
    init_distributed(backend="gloo")
    torch.manual_seed(0)
    m = models.build_model("mlp")
    o = AdamW(m.named_parameters(), lr=1e-3, state_bits=bits, mode=mode,
              grad_scale="mean", bucket_mb=0.05,
              no_decay=lambda n, p: p.dim() < 2)
    _train(m, o, steps=4, seed=rank)
    if mode != "async":
        cs = [None, None]
        dist.all_gather_object(cs, o.flat.param_checksum())
        assert len(set(cs)) == 1
    o.finish()
    assert torch.isfinite(_flat(m)).all()
    if rank == 0:
        open(out, "w").write("ok")


@pytest.mark.parametrize("mode,bits", [("replicated", 8), ("ps", 8),
                                       ("async", 8), ("replicated", 32)])
def test_two_ranks(tmp_path, mode, bits):
    """Every exchange mode; ranks that update alike round alike."""
    import socket
    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = tmp_path / "ok"
    mp.spawn(_worker, args=(port, mode, bits, str(out)), nprocs=2, join=True)
    assert out.read_text() == "ok"
