"""The path of windowed attention without a kernel: CPU, and other types and
head sizes on the GPU.  It keeps the kernels' promises."""

import pytest
import torch

from pytorch_ps_mpi_amd.ops.attn import fused_window_sdpa

GPU = pytest.param("cuda:0", marks=pytest.mark.gpu)


def _run(q, k, v, go, *args):
    x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    o = fused_window_sdpa(*x, *args)
    return [o.detach(), *torch.autograd.grad(o, x, go)]


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16,
                                   torch.bfloat16])
@pytest.mark.parametrize("bad", [torch.nan, torch.inf, -torch.inf])
def test_what_stands_behind_a_length_goes_nowhere(device, dtype, bad):
    """In q, k, v and in the output's gradient, by itself and all at once."""
    g = torch.Generator().manual_seed(0)
    B, N, D = 5, 9, 24  # a head size without a kernel
    lengths = [9, 4, 0, 1, 99]
    t = [torch.randn(B, h, N, D, generator=g).to(device, dtype)
         for h in (4, 2, 2, 4)]
    lens = torch.tensor(lengths, dtype=torch.int32, device=device)
    clean = []
    for x in t:
        c = x.clone()
        for b, n in enumerate(lengths):
            c[b, :, n:] = 0
        clean.append(c)
    want = _run(*clean, 3, 1, lens)
    for which in ((0,), (1,), (2,), (3,), (0, 1, 2, 3)):
        dirty = [c.clone() for c in clean]
        for i in which:
            for b, n in enumerate(lengths):
                dirty[i][b, :, n:] = bad
        got = _run(*dirty, 3, 1, lens)
        for x, y in zip(got, want):
            assert torch.equal(x, y), which
            for b, n in enumerate(lengths):
                assert (x[b, :, n:] == 0).all()


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,KV,N", [(2, 4, 2, 0), (0, 4, 2, 5), (0, 4, 2, 0),
                                      (2, 0, 2, 5)])
@pytest.mark.parametrize("padded", [False, True])
def test_empty(device, dtype, B, H, KV, N, padded):
    """No rows, no sequences or no query heads: an empty result with a graph
    behind it, zeros for keys that nothing looks at."""
    mk = lambda h: torch.randn(B, h, N, 64, device=device, dtype=dtype)  # noqa: E731
    lens = torch.ones(B, dtype=torch.int32, device=device) if padded else None
    o, dq, dk, dv = _run(mk(H), mk(KV), mk(KV), mk(H), 3, 1, lens)
    assert o.shape == dq.shape == (B, H, N, 64)
    assert dk.shape == dv.shape == (B, KV, N, 64)
    assert o.dtype == dtype and not dk.any() and not dv.any()


def test_heads_without_elements_are_refused():
    t = torch.empty(2, 2, 3, 0)
    with pytest.raises(ValueError, match="one element"):
        fused_window_sdpa(t, t, t, 3)


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_heads_are_stored_behind_the_rows(device, dtype):
    """The documented layout, whichever path computes: a view of it is what a
    projection of all heads reads."""
    q, k = (torch.randn(2, h, 7, 64, device=device, dtype=dtype)
            for h in (4, 2))
    o = fused_window_sdpa(q, k, k, 3)
    assert o.transpose(1, 2).is_contiguous()
    assert o.transpose(1, 2).view(2, 7, 4 * 64).data_ptr() == o.data_ptr()


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("padded", [False, True])
def test_autocast_leaves_the_sums_in_32_bits(device, dtype, padded):
    """The path promises scores and sums in 32 bits; autocast would turn its
    products into bf16 ones, forward and backward."""
    g = torch.Generator().manual_seed(0)
    t = [torch.randn(2, h, 9, 24, generator=g).to(device, dtype)
         for h in (4, 2, 2, 4)]
    lens = torch.tensor([9, 4], dtype=torch.int32,
                        device=device) if padded else None
    want = _run(*t, 3, 1, lens)
    with torch.autocast(t[0].device.type, dtype=torch.bfloat16):
        got = _run(*t, 3, 1, lens)
        x = [v.clone().requires_grad_() for v in t[:3]]
        o = fused_window_sdpa(*x, 3, 1, lens)
    later = [o.detach(), *torch.autograd.grad(o, x, t[3])]
    for a, b, c in zip(want, got, later):
        assert a.dtype == b.dtype and torch.equal(a, b) and torch.equal(a, c)
