"""Layer norm's backward pass on rows far from zero: lanes behind a row's end hold zeros, whose distance from the mean times rstd may pass fp32's range."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [20, 200, 520, 1000, 2051, 4104, 9000, 17000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_constant_row_far_from_zero(cols, dtype):
    """xhat of a constant row is 0, whatever its value: dx = rstd (g - mean g)."""
    say("layer_norm_backward large rows", cols, dtype)
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(5, cols, generator=g)
    x[1], x[3] = 2.0 ** 110, -2.0 ** 111                       # (multiples of a power of two up to 16 bits: sums and mean are exact)
    x, dy, w = x.to(dtype).cuda(), torch.randn(5, cols, generator=g).to(dtype).cuda(), (1 + 0.2 * torch.randn(cols, generator=g)).cuda()
    _, mean, rstd = Q.layer_norm(x, w, None, 1e-12)
    assert mean[1] == 2.0 ** 110 and mean[3] == -2.0 ** 111 and abs(rstd[1].item() * 1e-6 - 1) < 1e-6
    got = Q.layer_norm_backward(dy, x, mean, rstd, w, out_dtype=torch.float32)
    r = R.f64(rstd)[:, None]
    xhat = (R.f64(x) - R.f64(mean)[:, None]) * r
    assert (xhat[[1, 3]] == 0).all()
    ref, bound = R.norm_gradients(R.f64(dy), xhat, 2 * R.U * np.abs(xhat), r, R.f64(w))
    for name, t, want, e in zip(("dx", "dweight", "dbias"), got, ref, bound):
        R.check(t, want, R.stored(e, want, torch.float32), name)
