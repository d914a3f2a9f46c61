"""fused_gated_residual where a wave or block takes several rows (@gpu): the
next row on its way, sums carried from row to row, uneven numbers of rows.

A launch holds at most 4096 waves forward (8192 with both norms and 256 lanes
a row), 2048 backward, of 1 to 8 waves a row, so the sizes here are at least
two rounds of the one and four of the other, for each shape of a row.  The
bounds are those of test_gpu_join: a column's sum passes at most 9 rows of a
wave, 3 waves, 32 parts and 5 joins, within its 64 roundings.
"""

import pytest
import torch

from test_gpu_join import DEV, NAMES, _reference, _run
from test_join import call, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,D", [(9001, 72), (9001, 513), (9001, 768),
                                    (5003, 1032), (5003, 2056), (1301, 4104)])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate,kind", [("none", "rms"), ("channel", "layer"),
                                       ("sample", "rms"), ("token", "layer")])
def test_several_rows_a_block(dtype, rows, D, post, gate, kind):
    B = 3 if gate == "sample" else 1
    t = inputs(B, rows // B, D, dtype, gate, post, kind == "layer", seed=D)
    want, tol = _reference({n: None if v is None else v.to(DEV)
                            for n, v in t.items()}, 0.7, kind)
    got = _run(t, 0.7, kind)
    for n in want:
        assert got[n].shape == want[n].shape, n
        err = (got[n].double() - want[n]).abs()
        assert (err <= tol[n]).all(), (n, err.max(), (err / tol[n]).max())
