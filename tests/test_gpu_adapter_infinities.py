"""Infinities and NaN in factors, rows and gradients of adapters: what the formulas make no number of is infinite or NaN, and nothing else changes by a bit.  (Operands enter
the products as two or three numbers that add up to them, so that an infinity may come out as NaN: 0 times infinity, or infinities of both signs.)"""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROWS, ADAPTERS, K, N = 70, 3, 264, 200


def randn(*shape, seed, dtype, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def run(y, x, dy, A, B, groups, s, dx_dtype, grad):
    out, u = Q.add_adapters(y, x, A, B, groups, s, keep=True)
    dx, dA, dB = Q.add_adapters_backward(dy, x, u, A, B, groups, s, dx=torch.zeros(ROWS, K, dtype=dx_dtype, device="cuda"), grad_dtype=grad)
    return dict(u=u, out=out, dx=dx, dA=dA, dB=dB)


@pytest.mark.parametrize("rank", [1, 12, 16, 40, 128])
@pytest.mark.parametrize("dtype,wide", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("where", ["A", "B", "x", "dy", "y"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_they_stay_where_the_formulas_have_them(rank, dtype, wide, where, value):
    say("adapters infinities", rank, dtype, wide, where, value)
    t = dict(y=randn(ROWS, N, seed=1, dtype=wide), x=randn(ROWS, K, seed=2, dtype=dtype), dy=randn(ROWS, N, seed=3, dtype=dtype, scale=0.1),
             A=randn(ADAPTERS, rank, K, seed=4, dtype=dtype, scale=0.1), B=randn(ADAPTERS, rank, N, seed=5, dtype=dtype, scale=0.1))
    ids = torch.randint(-1, ADAPTERS, (ROWS,), generator=torch.Generator().manual_seed(6))
    ids[:4] = torch.tensor([1, 1, -1, 0])
    s, groups = torch.tensor([0.5, 1.0, 2.0], device="cuda"), Q.group_rows(ids.cuda(), ADAPTERS)
    clean = run(**t, groups=groups, s=s, dx_dtype=wide, grad=wide)
    at = (1, rank - 1, 7) if where in "AB" else (0, 7)
    t[where][at] = value
    got = run(**t, groups=groups, s=s, dx_dtype=wide, grad=wide)
    # no numbers: by the formulas in 64 bits, each out of what the kernels have in hand
    y, x, dy, A, B = (R.f64(t[k]) for k in ("y", "x", "dy", "A", "B"))
    want = {k: R.f64(v).copy() for k, v in clean.items()}
    with np.errstate(invalid="ignore"):
        for i in range(ADAPTERS):
            r = np.nonzero(ids.numpy() == i)[0]
            u, v = x[r] @ A[i].T, dy[r] @ B[i].T
            want["u"][r], want["out"][r], want["dx"][r] = u, y[r] + u @ B[i], v @ A[i]
            want["dA"][i], want["dB"][i] = v.T @ x[r], u.T @ dy[r]
        none = np.nonzero(ids.numpy() < 0)[0]
        want["out"][none] = y[none]
    for name in want:
        number = np.isfinite(want[name])
        assert np.array_equal(np.isfinite(R.f64(got[name])), number), name
        assert np.array_equal(R.f64(got[name])[number], R.f64(clean[name])[number]), name
        if np.isnan(value):
            assert np.isnan(R.f64(got[name])[~number]).all(), name
