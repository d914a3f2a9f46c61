"""Checkpoints of the optimizers: resume in other buckets, refusals."""

import pytest
import torch

from pytorch_ps_mpi_amd import SGD, Adam, AdamW, models
from test_adamw import _flat, _train


@pytest.mark.parametrize("cls,kw", [
    (AdamW, dict(state_bits=8, seed=5)), (AdamW, dict(state_bits=32)),
    (Adam, {}), (SGD, dict(momentum=0.9, dampening=0.5))])
@pytest.mark.parametrize("placed", [True, False])
def test_checkpoint_resumes_in_other_buckets(cls, kw, placed):
    """The number of a step (bias corrections, rounding bits, the first
    momentum) goes with the elements, wherever buckets are cut; checkpoints
    that do not hold the cuts included."""
    threads = torch.get_num_threads()
    torch.set_num_threads(1)  # several split the elementwise loops anew

    def made(mb):
        torch.manual_seed(0)
        m = models.build_model("mlp")
        return m, cls(m.named_parameters(), lr=1e-3, bucket_mb=mb, **kw)

    for first, then in ((50, 0.0001), (0.0001, 50), (0.0001, 0.0001)):
        m1, o1 = made(first)
        _train(m1, o1, steps=3)
        sd = o1.state_dict()
        if not placed:
            del sd["bucket_starts"]
        m2, o2 = made(then)
        o2.load_state_dict(sd)
        _train(m1, o1, steps=2, seed=4)
        _train(m2, o2, steps=2, seed=4)
        assert set(o2._bucket_apply_count) == set(range(len(o2.flat.buckets)))
        assert torch.equal(_flat(m1), _flat(m2))
    torch.set_num_threads(threads)


def test_checkpoint_of_uneven_buckets():
    """Counts that differ stay with their elements, and are refused where one
    bucket would need two of them, before anything has changed."""
    def made(mb):
        torch.manual_seed(0)
        m = models.build_model("mlp")
        return m, AdamW(m.named_parameters(), lr=1e-3, bucket_mb=mb)

    m1, o1 = made(0.0001)
    _train(m1, o1, steps=3)
    o1._bucket_apply_count[0] = 2
    sd = o1.state_dict()
    m2, o2 = made(0.0001)
    o2.load_state_dict(sd)
    assert o2._bucket_apply_count == o1._bucket_apply_count
    for take in (sd, {k: v for k, v in sd.items() if k != "bucket_starts"}):
        m3, o3 = made(50)
        before = _flat(m3)
        with pytest.raises(ValueError, match="updates"):
            o3.load_state_dict(take)
        assert torch.equal(_flat(m3), before) and o3._step_count == 0 \
            and not o3._bucket_apply_count
    fresh = made(50)[1].state_dict()
    o2.load_state_dict(fresh)
    assert not o2._bucket_apply_count


def test_refused_checkpoint_leaves_the_seed():
    """The seed chooses the rounding bits: a checkpoint that is refused, for
    whatever reason, must not change it."""
    o1 = AdamW(models.build_model("mlp").named_parameters(), seed=5,
               state_bits=8)
    sd = o1.state_dict()
    m = models.build_model("mlp")
    o2 = AdamW(m.named_parameters(), seed=9, state_bits=8)
    before = _flat(m)
    for bad in (dict(names=["another"]), dict(state_bits=32),
                dict(bucket_apply_count={0: 1}, bucket_starts=[0, 256])):
        with pytest.raises((AssertionError, ValueError)):
            o2.load_state_dict({**sd, **bad})
        assert o2.seed == 9 and torch.equal(_flat(m), before)
    o2.load_state_dict(sd)
    assert o2.seed == 5


@pytest.mark.parametrize("mb", [0, 0.0001, 50])
def test_buckets_without_elements(mb):
    """A parameter of no elements may be all of a bucket; no count is asked
    of it."""
    def made(mb):
        torch.manual_seed(0)
        named = [("none", torch.nn.Parameter(torch.zeros(0))),
                 ("a", torch.nn.Parameter(torch.randn(300))),
                 ("empty", torch.nn.Parameter(torch.zeros(0, 3))),
                 ("b", torch.nn.Parameter(torch.randn(20)))]
        return AdamW(named, lr=1e-2, bucket_mb=mb)

    def train(o, steps):
        for _ in range(steps):
            o.zero_grad()
            o.flat.flat_grad.copy_(o.flat.flat_param)
            o.step()

    o1 = made(0)
    train(o1, 3)
    o2 = made(mb)
    o2.load_state_dict(o1.state_dict())
    train(o2, 1)
    o3 = made(50)
    o3.load_state_dict(o2.state_dict())
    train(o1, 3)
    train(o3, 2)
    assert torch.equal(o1.flat.master, o3.flat.master)
