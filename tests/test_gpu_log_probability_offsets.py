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
    """log p, entropy, and the bounds of log S and of the entropy.  An exponential's argument is x - max, rounded, times log2 e, rounded (U |d| each on the exponential), its value is
    off by a last place or two; a lane adds eight of every 2048 columns one after the other, puts its sums right no more than once for every octet (twice the largest
    |d| in U, and three roundings, each time that the maximum grows: all these factors together span no more than the largest |d|), 20 exchanges
    behind that."""
    d = x - x.max(-1, keepdims=True)
    e = np.exp(d)
    S = e.sum(-1, keepdims=True)
    p, near = e / S, np.where(e > 0, d, 0.0)
    octets = x.shape[-1] / 2048 + 2
    each = R.U * (2 * np.abs(near) + 4 + 11 * octets + 40 + 4 * np.abs(near).max(-1, keepdims=True))
    e_S, T = (p * each).sum(-1, keepdims=True), -(p * near).sum(-1, keepdims=True)
    lp = d - np.log(S)
    e_H = e_S * (1 + T) + (p * np.abs(near) * each).sum(-1, keepdims=True) + 4 * R.U * (np.log(S) + T)
    return lp, -(p * np.where(e > 0, lp, 0.0)).sum(-1), e_S + 3 * R.U * np.log(S), e_H


def check_forward(x, tokens, top):
    logp, entropy, lse, values, indices = Q.log_probabilities(x, tokens, top)
    X, T, rows = R.f64(x), tokens.cpu().numpy(), np.arange(len(x))
    lp, H, e_l, _ = statistics(X)
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


def check_gradients(x, tokens, entropy, lse, a, b, out_dtype=None):
    """Up to FAR, log p = x - lse has the rounding of lse, beyond it nothing but its own (an absolute error of log p is a relative one of p)."""
    dx = Q.log_probabilities_backward(x, tokens, lse, entropy, a, b, out_dtype)
    X, T, rows = R.f64(x), tokens.cpu().numpy(), np.arange(len(x))
    A, B, z = R.f64(a)[:, None], R.f64(b)[:, None], R.f64(lse)[:, None]
    lp, H, e_l, e_H = statistics(X)
    p, away, H = np.exp(lp), np.abs(X - X.max(-1, keepdims=True)), H[:, None]
    near = np.where(p > 0, lp, 0.0)
    e_lp = e_l + R.U * (np.where(p > 0, away, 0.0) + 2 * np.abs(near)) + np.where(np.abs(z) <= FAR, R.U * np.abs(z), 0.0)
    inner = A + B * (near + H)
    ref = -p * inner
    ref[rows, T] += A[:, 0]
    bound = p * (np.abs(inner) * (e_lp + R.U * (2 * np.abs(near) + 4)) + 4 * R.U * (np.abs(A) + np.abs(B) * (np.abs(near) + H)) + np.abs(B) * (e_lp + e_H)) + 2 * R.U * np.abs(ref)
    bound[rows, T] += 2 * R.U * np.abs(A[:, 0])
    R.check(dx, ref, R.stored(bound, ref, dx.dtype), "dlogits")
    return dx, bound.sum(-1)


@pytest.mark.parametrize("cols", [40, 1000, 5003, 70001])
@pytest.mark.parametrize("dtype,out_dtype", [(F32, None), (BF16, None), (F16, None), (BF16, F32)])
@pytest.mark.parametrize("many", [False, True])
def test_gradients_of_rows_far_from_zero(cols, dtype, out_dtype, many):
    """A row's gradient adds up to nothing, whatever p is: a (1 - 1) - b sum of p (log p + entropy)."""
    say("log_probabilities_backward far from zero", cols, dtype, out_dtype, many)
    x, tokens, _ = rows_far_from_zero(cols, dtype)
    again = 150 if many else 1
    x, tokens = x.repeat(again, 1), tokens.repeat(again)
    _, entropy, lse = Q.log_probabilities(x, tokens)
    a, b = torch.linspace(-1, 2, len(x), device="cuda"), torch.linspace(1.5, -1, len(x), device="cuda")
    with np.errstate(invalid="ignore"):
        dx, bound = check_gradients(x, tokens, entropy, lse, a, b, out_dtype)
    if dx.dtype == F32:
        assert (np.abs(R.f64(dx).sum(-1)) <= bound + R.U * np.abs(R.f64(dx)).sum(-1)).all()


@pytest.mark.parametrize("offset", [0, 120, 127.9, 128.1, 500, -127.9, -128.1, 7e4])
def test_gradients_on_both_sides_of_the_bound(offset):
    """Rows whose lse lies just inside and just outside of what x - lse serves, side by side with a masked row and one that asks for nothing."""
    say("log_probabilities_backward bound", offset)
    cols = 3001
    x = torch.randn(6, cols, generator=torch.Generator().manual_seed(3)).cuda()
    x += offset - torch.logsumexp(x, 1, keepdim=True)
    x[2, ::2] = float("-inf")
    x[4] = float("-inf")
    tokens = torch.tensor([0, 5, 7, 9, 11, cols - 1], device="cuda")
    a, b = torch.linspace(-1, 2, 6, device="cuda"), torch.linspace(1.5, -1, 6, device="cuda")
    _, entropy, lse = Q.log_probabilities(x, tokens)
    keep = torch.tensor([0, 1, 2, 3, 5], device="cuda")
    whole = Q.log_probabilities_backward(x, tokens, lse, entropy, a, b)
    assert (whole[4] == 0).all()
    with np.errstate(invalid="ignore"):
        dx, _ = check_gradients(x[keep], tokens[keep], entropy[keep], lse[keep], a[keep], b[keep])
    assert torch.equal(dx, whole[keep])
    tokens[3] = -100
    unasked = Q.log_probabilities_backward(x, tokens, lse, entropy, a, b)
    zero = a.clone()
    zero[3] = 0
    tokens[3] = 9
    assert torch.equal(unasked, Q.log_probabilities_backward(x, tokens, lse, entropy, zero, b))


def test_gradients_far_from_zero_in_a_graph():
    """The graph takes what lies there when it is replayed, rows near and far."""
    say("log_probabilities_backward far captured")
    x, tokens, a = torch.zeros(6, 70000, device="cuda"), torch.tensor([0, 5, 7, 9, 11, 13], device="cuda"), torch.ones(6, device="cuda")

    def both():
        _, H, lse = Q.log_probabilities(x, tokens)
        return H, lse, Q.log_probabilities_backward(x, tokens, lse, H, a, a)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed, offset in ((1, 0.0), (2, 1e4), (3, -1e9), (4, 3.0)):
        x.copy_(torch.randn(6, 70000, generator=torch.Generator().manual_seed(seed)) + torch.tensor([offset, 0, offset, 0, 0, 1e3])[:, None])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, both()))


@pytest.mark.parametrize("cols", [30, 5000])
@pytest.mark.parametrize("bonus", [None, 0.0, 1.0])
def test_padding_rows_have_no_gradient_whatever_they_hold(cols, bonus):
    """Rows that ask for nothing, with NaN and infinities in them: no gradient comes of their log p, and none of an entropy that has no gradient."""
    say("log_probabilities_backward padding", cols, bonus)
    x, tokens = torch.randn(6, cols, generator=torch.Generator().manual_seed(1)).cuda(), torch.tensor([3, -100, -100, cols, 4, -100], device="cuda")
    x[1], x[2, 5], x[3, 0] = float("nan"), float("inf"), float("nan")
    _, entropy, lse = Q.log_probabilities(x, tokens)
    a, b = torch.ones(6, device="cuda"), None if bonus is None else torch.zeros(6, device="cuda")
    a[3] = float("nan")
    if bonus:
        b[0], b[5] = bonus, bonus
    dx = Q.log_probabilities_backward(x, tokens, lse, entropy if bonus is not None else None, a, b)
    assert (dx[1:4] == 0).all() and torch.isfinite(dx).all()
    assert ((dx[5] != 0).any() if bonus else (dx[5] == 0).all()) and (dx[0] != 0).any() and (dx[4] != 0).any()
    if bonus:
        b[1] = bonus                                       # (an entropy that is asked for is NaN, and so is its gradient)
        assert torch.isnan(Q.log_probabilities_backward(x, tokens, lse, entropy, a, b)[1]).all()
