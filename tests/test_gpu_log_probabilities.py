"""Log probabilities, entropies and most probable tokens, and their gradients, against the formulas in 64 bits."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import language_ref as L
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def logits_of(rows, cols, dtype, seed, gap=0, offset=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(rows, cols, generator=g) * spread
    room = torch.full((offset + rows * (cols + gap) + 16,), float("nan"), dtype=dtype, device="cuda")
    t = room[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
    t.copy_(v.to(dtype))
    return t


def tokens_of(rows, cols, seed, dtype=torch.int64):
    t = torch.randint(0, cols, (rows,), generator=torch.Generator().manual_seed(seed))
    t[rows // 2:rows // 2 + 1] = -100
    if rows > 3:
        t[1], t[2] = cols, cols - 1
    return t.to(dtype).cuda()


def check(x, tokens, top):
    out = Q.log_probabilities(x, tokens, top)
    assert len(out) == (5 if top else 3)
    cols = x.shape[-1]
    X, T = R.f64(x).reshape(-1, cols), tokens.cpu().numpy().reshape(-1)
    (lp, H, lse), (e_lp, e_H, e_lse) = L.log_probabilities(X)
    rows = np.arange(len(X))
    asked = (T >= 0) & (T < cols)
    at = np.where(asked, T, 0)
    want = np.where(asked, lp[rows, at], 0.0)
    for got, ref, bound, name in ((out[0], want, e_lp[rows, at] + R.U * np.abs(want), "logp"), (out[1], H, e_H + R.U * np.abs(H), "entropy"),
                                  (out[2], lse, e_lse + R.U * np.abs(lse), "lse")):
        assert got.dtype == F32 and got.shape == x.shape[:-1]
        got = R.f64(got).reshape(-1)
        same = np.isneginf(ref)
        assert np.array_equal(np.isneginf(got), same), name
        R.check(torch.from_numpy(got[~same]), ref[~same], bound[~same], name)
    if top:
        order = np.argsort(-X, axis=1, kind="stable")[:, :top]
        assert out[4].dtype == torch.int64 and out[3].shape == out[4].shape == (*x.shape[:-1], top)
        assert np.array_equal(out[4].cpu().numpy().reshape(-1, top), order)
        ref, bound = np.take_along_axis(lp, order, 1), np.take_along_axis(e_lp, order, 1)
        got, gone = R.f64(out[3]).reshape(-1, top), np.isneginf(ref)
        assert np.array_equal(np.isneginf(got), gone)
        R.check(torch.from_numpy(got[~gone]), ref[~gone], bound[~gone] + R.U * np.abs(ref[~gone]), "values")
    return out


SIZES = [(1, 1), (2, 3), (5, 8), (3, 33), (7, 100), (1, 500), (64, 512), (3, 2047), (2, 2048), (9, 2049), (300, 1000), (4, 5003), (2, 16384), (1, 50001), (8, 131072),
         (1100, 4099), (2, 262147)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype,top", [(F32, 20), (BF16, 5), (F16, 0), (BF16, 32), (F32, 1)])
def test_forward(rows, cols, dtype, top):
    say("log_probabilities", rows, cols, dtype, top)
    check(logits_of(rows, cols, dtype, rows + cols), tokens_of(rows, cols, 2, torch.int32 if top == 5 else torch.int64), min(top, cols))


@pytest.mark.parametrize("cols", [12, 300, 2500, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties_go_to_the_lowest_token(cols, dtype):
    """Rows of one value, of two, of rising and of falling values, zeros of both signs; more equal values than there is room for candidates."""
    say("log_probabilities ties", cols, dtype)
    x = torch.zeros(7, cols, device="cuda", dtype=dtype)
    x[1] = torch.arange(cols, device="cuda") % 2
    x[2] = torch.arange(cols, device="cuda") / cols
    x[3] = -torch.arange(cols, device="cuda") / cols
    x[4, ::3] = -0.0
    x[5, :: max(1, cols // 7)] = 3.0
    x[6] = (torch.arange(cols, device="cuda") // 8 % 256 < 3).to(dtype)          # the columns of three threads hold all of the largest
    check(x, tokens_of(7, cols, 3), min(32, cols))


@pytest.mark.parametrize("rows,cols", [(3, 40000), (1100, 20000)])
@pytest.mark.parametrize("groups", [31, 8, 1])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_candidates_than_there_is_room_for(rows, cols, groups, dtype):
    """All that is large lies in the columns of a few threads, so that the first bound lets thousands of elements through; in rising order every one is above those before."""
    say("log_probabilities candidates", rows, cols, groups, dtype)
    x = logits_of(rows, cols, dtype, 4) - 20
    own = torch.arange(cols, device="cuda") // 8 % 256 < 4 * groups
    x[:, own] += 20
    x[1, own] = torch.arange(int(own.sum()), device="cuda").to(dtype) / 1024
    x[2, own] = 3.0
    check(x, tokens_of(rows, cols, 5), 32)


@pytest.mark.parametrize("cols", [40, 3000, 70001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_masks(cols, dtype):
    """-inf and the type's lowest value: over half of a row, over all but one column, over all of it."""
    say("log_probabilities masks", cols, dtype)
    x = logits_of(9, cols, dtype, 5)
    out = torch.rand(cols, generator=torch.Generator().manual_seed(6)) < 0.5
    out[0], out[1] = True, False
    out = out.cuda()
    low = torch.finfo(dtype).min
    x[0, out] = -INF
    x[1, out] = low
    x[2] = -INF
    x[3] = low
    x[4, 1:] = -INF
    x[5, :-1] = low
    x[6, :cols // 2] = -INF
    x[6, cols // 2:] = low
    x[7] = -INF
    x[7, cols - 3:] = low
    tokens = torch.tensor([1, 1, 0, 2, 0, cols - 1, 0, cols - 1, 5], device="cuda")
    got = check(x, tokens, 20)
    assert got[2][2] == -INF and got[0][2] == -INF and got[1][2] == 0
    _, H, lse = got[:3]
    a, b = torch.linspace(-1, 1, 9, device="cuda"), torch.linspace(1, -2, 9, device="cuda")
    check_backward(x, tokens, lse, H, a, b)
    assert (Q.log_probabilities_backward(x, tokens, lse, H, a, b)[2] == 0).all()


@pytest.mark.parametrize("cols", [30, 5000, 80000])
def test_infinities_and_nans_stay_in_their_rows(cols):
    say("log_probabilities special values", cols)
    x, tokens = logits_of(5, cols, F32, 7), torch.tensor([3, 2, -1, 4, 5], device="cuda")
    clean = Q.log_probabilities(x, tokens, 5)
    x[1, cols // 2] = float("nan")
    x[3, 7] = INF
    got = Q.log_probabilities(x, tokens, 5)
    for i in (0, 2, 4):
        assert all(torch.equal(a[i], b[i]) for a, b in zip(got, clean))
    for i in (1, 3):
        assert torch.isnan(got[0][i]) and torch.isnan(got[1][i]) and torch.isnan(got[2][i]) and torch.isnan(got[3][i]).all()
    assert got[4][3, 0] == 7 and (got[4] >= 0).all() and (got[4] < cols).all()
    dx = Q.log_probabilities_backward(x, tokens, got[2], got[1], torch.ones(5, device="cuda"), torch.ones(5, device="cuda"))
    assert torch.isnan(dx[1]).all() and torch.isnan(dx[3]).all() and torch.isfinite(dx[[0, 2, 4]]).all()


@pytest.mark.parametrize("shape,gap,offset", [((5, 1000), 7, 1), ((3, 5003), 1, 3), ((2, 3, 700), 0, 0), ((2, 2, 2, 90), 6, 0), ((900,), 0, 1)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_addresses_and_dimensions(shape, gap, offset, dtype):
    say("log_probabilities strides", shape, gap, offset, dtype)
    rows = int(np.prod(shape[:-1]))
    x = logits_of(rows, shape[-1], dtype, 8, gap, offset)
    x = x[0] if len(shape) == 1 else x.unflatten(0, shape[:-1])
    tokens = tokens_of(rows, shape[-1], 9).reshape(shape[:-1])
    out = check(x, tokens, 3)
    a = torch.randn(shape[:-1], generator=torch.Generator().manual_seed(10)).cuda()
    check_backward(x, tokens, out[2], out[1], a, 2 * a)


# ---- backward
def check_backward(x, tokens, lse, H, a, b, out_dtype=None):
    dx = Q.log_probabilities_backward(x, tokens, lse, H, a, b, out_dtype)
    cols = x.shape[-1]
    flat = lambda t: R.f64(t).reshape(-1)  # noqa: E731
    ref, bound = L.logit_gradients(R.f64(x).reshape(-1, cols), tokens.cpu().numpy().reshape(-1).astype(np.int64), flat(lse), flat(lse) * 0 if H is None else flat(H), flat(a),
                                   0 * flat(a) if b is None else flat(b))
    assert dx.dtype == (out_dtype or x.dtype) and dx.shape == x.shape
    R.check(dx, ref, R.stored(bound, ref, dx.dtype), "dlogits")
    return dx


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype,out,entropy", [(F32, None, True), (BF16, None, True), (F16, None, False), (F32, BF16, True), (BF16, F32, False)])
def test_backward(rows, cols, dtype, out, entropy):
    say("log_probabilities_backward", rows, cols, dtype, out, entropy)
    x, tokens = logits_of(rows, cols, dtype, rows + cols), tokens_of(rows, cols, 11)
    _, H, lse = Q.log_probabilities(x, tokens)
    g = torch.Generator().manual_seed(12)
    a, b = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    check_backward(x, tokens, lse, H if entropy else None, a, b if entropy else None, out)


@pytest.mark.parametrize("cols", [17, 1000])
def test_backward_against_differences(cols):
    say("log_probabilities differences", cols)
    x, tokens = logits_of(6, cols, F32, 13), tokens_of(6, cols, 14)
    _, H, lse = Q.log_probabilities(x, tokens)
    a, b = torch.linspace(-1, 1, 6, device="cuda"), torch.linspace(0.5, -2, 6, device="cuda")
    dx = R.f64(Q.log_probabilities_backward(x, tokens, lse, H, a, b))
    X, T, A, B = R.f64(x), tokens.cpu().numpy(), R.f64(a), R.f64(b)
    asked = (T >= 0) & (T < cols)

    def value(X):
        (lp, H, _), _ = L.log_probabilities(X)
        return (np.where(asked, A, 0) * lp[np.arange(6), np.where(asked, T, 0)]).sum() + (B * H).sum()

    rng = np.random.default_rng(2)
    for _ in range(8):
        d, step = rng.standard_normal(X.shape), 1e-5
        want = (value(X + step * d) - value(X - step * d)) / (2 * step)
        assert abs((dx * d).sum() - want) <= 1e-4 * np.sqrt((dx ** 2).sum())


def test_no_rows():
    say("log_probabilities no rows")
    x, t = torch.empty(0, 100, dtype=BF16, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    out = Q.log_probabilities(x, t, 4)
    assert out[0].shape == (0,) and out[4].shape == (0, 4)
    assert Q.log_probabilities_backward(x, t, out[2], out[1], out[0]).shape == (0, 100)


@pytest.mark.parametrize("rows,cols", [(4, 100000), (900, 6000)])
def test_the_same_bits_again_and_on_another_stream(rows, cols):
    say("log_probabilities again", rows, cols)
    x, tokens = logits_of(rows, cols, BF16, 15), tokens_of(rows, cols, 16)
    first = Q.log_probabilities(x, tokens, 20)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = Q.log_probabilities(x, tokens, 20)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_a_captured_pass():
    say("log_probabilities captured")
    x, tokens, a = logits_of(6, 70000, BF16, 17), tokens_of(6, 70000, 18), torch.ones(6, device="cuda")

    def both():
        logp, H, lse, v, i = Q.log_probabilities(x, tokens, 8)
        return logp, H, lse, v, i, Q.log_probabilities_backward(x, tokens, lse, H, a, a)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in (19, 20, 21):
        x.copy_(logits_of(6, 70000, BF16, seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, both()))


def test_through_ctypes(monkeypatch):
    say("log_probabilities ctypes")
    x, tokens = logits_of(6, 1000, BF16, 22).view(2, 3, 1000), tokens_of(6, 1000, 23).view(2, 3)

    def both():
        out = Q.log_probabilities(x, tokens, 5)
        return (*out, *Q.log_probabilities(x, tokens), Q.log_probabilities_backward(x, tokens, out[2], out[1], out[0], out[1], F32),
                Q.log_probabilities_backward(x, tokens, out[2], None, out[0]))

    want = both()
    monkeypatch.setattr(Q.ops, "_native_module", False)
    assert all(torch.equal(a, b) for a, b in zip(want, both()))


def test_offsets_beyond_32_bits():
    say("log_probabilities offsets")
    rows, cols = 65600, 65600
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    tail, t = logits_of(3, cols, BF16, 24), torch.zeros(rows, dtype=torch.int64, device="cuda")
    x[-3:] = tail
    t[-3:] = torch.tensor([5, cols - 1, 77], device="cuda")
    out, want = Q.log_probabilities(x, t, 4), Q.log_probabilities(tail.repeat(400, 1), t[-3:].repeat(400), 4)
    assert all(torch.equal(a[-3:], b[:3]) for a, b in zip(out, want))
    dx = Q.log_probabilities_backward(x, t, out[2], out[1], out[0], out[1])
    assert torch.equal(dx[-3:], Q.log_probabilities_backward(tail, t[-3:], out[2][-3:], out[1][-3:], out[0][-3:], out[1][-3:]))
