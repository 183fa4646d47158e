"""Layer norm's backward pass on rows of millions of columns: the parameters' sums of every column."""
import pytest
import torch

import qgemm_amd as Q
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(3, (1 << 21) + 37), (2, (1 << 22) - 1), (1, (1 << 28) + 5), (600, (1 << 20) + 9)])
def test_sums_of_every_column(rows, cols):
    say("layer_norm_backward wide rows", rows, cols)
    g = torch.Generator(device="cuda").manual_seed(cols)
    dy, x = (torch.randint(-8, 9, (rows, cols), generator=g, device="cuda", dtype=torch.int8).bfloat16() for _ in range(2))
    mean, rstd, w = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda"), torch.ones(cols, device="cuda")
    dx, dw, db = Q.layer_norm_backward(dy, x, mean, rstd, w, out_dtype=torch.float32)
    # (whole numbers: the columns' sums are exact)
    assert torch.equal(db, dy.float().sum(0)) and torch.equal(dw, (dy.float() * x.float()).sum(0))
    for row in range(0, rows, max(1, rows // 3)):
        d, v = dy[row].double(), x[row].double()
        a, b = d.mean(), (d * v).mean()
        # a lane adds up every 256th octet, one after the other
        adds = (cols / 2048 + 64) * R.U
        e = adds * d.abs().mean() + adds * (d * v).abs().mean() * 8 + 4 * R.U * (8 + a.abs() + 8 * b.abs())
        assert (dx[row].double() - (d - a - v * b)).abs().max() <= e
