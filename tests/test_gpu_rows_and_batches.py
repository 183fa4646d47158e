"""A row by itself and the same row in a large batch: what is the same bit for bit, and what is so within the bounds of its sums."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import language_ref as L
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [500, 8192, 8200, 50001, 131072])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_log_probabilities(cols, dtype):
    """Few rows are split, many are not: the sums are added in another order.  The tokens are the same, and each number lies within its bound on either side."""
    say("a row alone and in a batch", cols, dtype)
    g = torch.Generator().manual_seed(cols)
    row, t = (torch.randn(1, cols, generator=g) * 3).to(dtype).cuda(), torch.tensor([cols // 3], device="cuda")
    alone, many = Q.log_probabilities(row, t, 20), Q.log_probabilities(row.repeat(1100, 1), t.repeat(1100), 20)
    for m in many:
        assert torch.equal(m, m[:1].expand_as(m))
    assert torch.equal(alone[4], many[4][:1])
    (lp, _, lse), (e_lp, e_H, e_lse) = L.log_probabilities(R.f64(row))
    at = R.f64(alone[4]).astype(np.int64)[0]
    e = np.concatenate([e_lp[0, [cols // 3]] + R.U * np.abs(lp[0, cols // 3]), e_H, e_lse + R.U * np.abs(lse), e_lp[0, at] + R.U * np.abs(lp[0, at])])
    flat = lambda out: np.concatenate([R.f64(v[:1]).reshape(-1) for v in out[:4]])  # noqa: E731
    assert (np.abs(flat(alone) - flat(many)) <= 2 * e + 2 * R.U * np.abs(flat(alone))).all()
    # the gradient's bits are the same: every element is computed out of its own logit and its row's numbers
    a = torch.ones(1, device="cuda")
    for h in (None, a):
        one = Q.log_probabilities_backward(row, t, alone[2], alone[1], a, h)
        all_ = Q.log_probabilities_backward(row.repeat(1100, 1), t.repeat(1100), alone[2].repeat(1100), alone[1].repeat(1100), a.repeat(1100), None if h is None else h.repeat(1100))
        assert torch.equal(all_, one.expand_as(all_))


@pytest.mark.parametrize("cols", [100, 7168, 20000])
def test_rms_norm(cols):
    say("a row of the norm alone and in a batch", cols)
    x = torch.randn(1, cols, generator=torch.Generator().manual_seed(cols)).bfloat16().cuda()
    w = torch.linspace(0.5, 1.5, cols, device="cuda")
    alone, many = Q.rms_norm(x, w, codes=torch.int8), Q.rms_norm(x.repeat(3000, 1), w, codes=torch.int8)
    assert all(torch.equal(m, a.expand_as(m)) for a, m in zip(alone, many))
