"""Log probabilities, top values and gradients of rows whose numbers lie far from zero: masked throughout with a finite number, or with a common offset, so that
log sum exp keeps few or none of the bits of log S.  The reference never forms it: log p = (x - max) - log S."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FAR = 128.0                                                # up to here the gradient takes log p = x - lse


def statistics(x):
    """log p, entropy, and the bound of log S.  An exponential's argument is x - max, rounded, times log2 e, rounded (U |d| each on the exponential), its value is
    off by a last place or two; a lane adds eight of every 2048 columns one after the other, puts its sums right no more than once for every octet (twice the largest
    |d| in U, and three roundings, each time that the maximum grows: all these factors together span no more than the largest |d|), 20 exchanges
    behind that."""
    d = x - x.max(-1, keepdims=True)
    e = np.exp(d)
    S = e.sum(-1, keepdims=True)
    p, near = e / S, np.where(e > 0, d, 0.0)
    octets = x.shape[-1] / 2048 + 2
    each = R.U * (2 * np.abs(near) + 4 + 11 * octets + 40 + 4 * np.abs(near).max(-1, keepdims=True))
    e_S = (p * each).sum(-1, keepdims=True)
    lp = d - np.log(S)
    return lp, -(p * np.where(e > 0, lp, 0.0)).sum(-1), e_S + 3 * R.U * np.log(S)


def check_forward(x, tokens, top):
    logp, entropy, lse, values, indices = Q.log_probabilities(x, tokens, top)
    X, T, rows = R.f64(x), tokens.cpu().numpy(), np.arange(len(x))
    lp, H, e_l = statistics(X)
    away = np.abs(X - X.max(-1, keepdims=True))            # (x - max is rounded, and so is the difference of that and log S)
    bound = e_l + R.U * (away + 2 * np.abs(lp))
    R.check(logp, lp[rows, T], bound[rows, T], "logp")
    order = np.argsort(-X, axis=1, kind="stable")[:, :top]
    assert np.array_equal(indices.cpu().numpy(), order)
    want, bound, values = np.take_along_axis(lp, order, 1), np.take_along_axis(bound, order, 1), R.f64(values)
    gone = np.isneginf(want)                               # (what -inf masks)
    assert np.array_equal(np.isneginf(values), gone)
    R.check(torch.from_numpy(values[~gone]), want[~gone], bound[~gone], "values")
    return entropy, lse


def rows_far_from_zero(cols, dtype):
    """One for each way in which a row comes to lie far away, and how many columns of it are left where it is a mask."""
    g = torch.Generator().manual_seed(cols)
    low, noise = torch.finfo(dtype).min, torch.randn(8, cols, generator=g)
    x = noise.clone()
    x[0] = low
    x[1] = -1e4
    x[2, :cols // 2], x[2, cols // 2:] = float("-inf"), low
    x[3], x[3, cols - 3:] = float("-inf"), low
    x[4] = noise[4] + (1e5 if dtype != F16 else 6e4)
    x[5] = noise[5] - (1e5 if dtype != F16 else 6e4)
    x[6] = noise[6] + 200
    x[7] = -1e9 if dtype != F16 else -6e4
    left = {0: cols, 1: cols, 2: cols - cols // 2, 3: 3, 7: cols}
    return x.to(dtype).cuda(), torch.tensor([1, cols - 1, cols // 2, cols - 2, 0, cols // 3, 2, cols // 2], device="cuda"), left


@pytest.mark.parametrize("cols", [40, 1000, 5003, 70001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("many", [False, True])
def test_rows_far_from_zero(cols, dtype, many):
    """By themselves, which splits a long row, and among so many that it is not."""
    say("log_probabilities far from zero", cols, dtype, many)
    x, tokens, left = rows_far_from_zero(cols, dtype)
    again = 150 if many else 1
    with np.errstate(invalid="ignore"):
        entropy, _ = check_forward(x.repeat(again, 1), tokens.repeat(again), 20)
    logp = R.f64(Q.log_probabilities(x, tokens)[0])
    for row, n in left.items():
        assert abs(logp[row] + np.log(n)) <= 1e-5 * np.log(n) and abs(entropy[row].item() - np.log(n)) <= 1e-5 * np.log(n), (row, logp[row])
