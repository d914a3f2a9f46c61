"""Parts of an 8-bit state."""

import pytest
import torch

from pytorch_ps_mpi_amd import ops


def test_parts():
    st = ops.State8.zeros(700, True)
    st.codes.copy_(torch.arange(700) % 128)
    st.scales.copy_(torch.tensor([1.0, 2.0, 4.0]))
    whole = st.values()
    for a, b in ((0, 700), (0, 256), (256, 512), (256, 700), (512, 700),
                 (0, 0), (512, 512)):
        assert torch.equal(st.span(a, b).values(), whole[a:b])


@pytest.mark.parametrize("start,end", [
    (-256, 700), (0, 768), (512, 256), (-512, -256), (0, -256), (1024, 1024),
    (100, 700), (0, 100)])
def test_parts_that_do_not_exist_are_refused(start, end):
    """A negative start would count codes and scales from different ends."""
    with pytest.raises(ValueError):
        ops.State8.zeros(700, True).span(start, end)
