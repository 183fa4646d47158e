"""Layer norm, forward and backward, against the formulas in 64 bits, at the sizes, strides and values where it can go wrong."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, F8 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
EPS = 1e-5


def rows_of(shape, dtype, seed, gap=0, offset=0, mean=0.3):
    """Values with channels of different size and rows off centre, in rows `gap` elements longer than they need be."""
    g = torch.Generator().manual_seed(seed)
    rows, cols = int(np.prod(shape[:-1])), shape[-1]
    v = torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g)) + mean * torch.randn(rows, 1, generator=g)
    room = torch.full((offset + rows * (cols + gap) + 16,), float("nan"), dtype=dtype, device="cuda")
    t = room[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
    t.copy_(v.to(dtype))
    return t if len(shape) == 2 else t.view(shape) if gap == 0 else t.unflatten(0, shape[:-1])


def params_of(cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return ((1 + 0.2 * torch.randn(cols, generator=g)).to(dtype).cuda(), (0.1 * torch.randn(cols, generator=g)).to(dtype).cuda())


def check_forward(x, w, b, eps=EPS, out_dtype=None, keep=None):
    out = Q.layer_norm(x, w, b, eps, out_dtype=out_dtype, keep=keep)
    y, mean, rstd = out[:3]
    cols = x.shape[-1]
    assert y.shape == x.shape and y.dtype == (out_dtype or x.dtype) and mean.shape == rstd.shape == x.shape[:-1]
    (ry, rm, rr, rx), (ey, em, er, ex) = R.norm(R.f64(x).reshape(-1, cols), None if w is None else R.f64(w), None if b is None else R.f64(b), eps)
    R.check(mean, rm, em + R.U * np.abs(rm), "mean")
    R.check(rstd, rr, er, "rstd")
    R.check(y, ry, R.stored(ey, ry, y.dtype), "y")
    if keep is not None:
        q, s = out[3:]
        assert q.dtype == keep and q.shape == x.shape and s.shape == (*x.shape[:-1], -(-cols // 128))
        # the scale of the exact xhat, or its neighbour where xhat's error reaches over the edge
        got, top = R.f64(s).reshape(rx.shape[0], -1), np.abs(R.blocks(rx)).max(-1)
        wide = np.broadcast_to(ex, rx.shape).reshape(rx.shape)
        slack = np.abs(R.blocks(wide)).max(-1)
        assert (np.exp2(np.rint(np.log2(got))) == got).all()
        assert (top - slack <= R.LARGEST[keep] * got).all()
        assert ((top + slack > R.LARGEST[keep] * got / 2) | ((got == 1) & (top <= slack))).all()
        v = R.values(q, s)
        full = np.repeat(got, 128, 1)[:, :cols]
        half = full / 2 if keep == I8 else np.maximum(np.abs(rx) * 2.0 ** -4, full * 2.0 ** -10)
        R.check(torch.from_numpy(v), rx, half * (1 + 1e-6) + 2 * ex, "kept")
        assert np.abs(R.f64(q)).max() <= R.LARGEST[keep]
    return out


SIZES = [(1, 1), (3, 5), (2, 8), (5, 64), (300, 64), (17, 127), (513, 128), (9, 130), (100, 257), (33, 512), (5, 1000), (3, 1024), (64, 2048), (7, 2056),
         (5, 3001), (3, 4104), (2, 7168), (600, 7168), (3, 8200), (2, 16384), (2, 16392), (1, 20001), (2, 40000)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype,params,keep", [(BF16, F32, I8), (F16, F16, F8), (F32, F32, None), (BF16, BF16, None), (F32, BF16, I8)])
def test_forward(rows, cols, dtype, params, keep):
    say("layer_norm", rows, cols, dtype, params, keep)
    check_forward(rows_of((rows, cols), dtype, rows + cols), *params_of(cols, params, 3), keep=keep)


@pytest.mark.parametrize("cols", [64, 128, 1000, 3001, 7168])
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False)])
def test_forward_without_parameters(cols, weight, bias):
    say("layer_norm without parameters", cols, weight, bias)
    w, b = params_of(cols, F32, 5)
    check_forward(rows_of((40, cols), BF16, 6), w if weight else None, b if bias else None, keep=I8)


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [96, 1001, 5000])
def test_forward_into_another_type(cols, out_dtype):
    say("layer_norm out_dtype", cols, out_dtype)
    check_forward(rows_of((9, cols), F16, 8), *params_of(cols, F16, 9), out_dtype=out_dtype)


@pytest.mark.parametrize("shape,gap,offset", [((7, 128), 3, 1), ((70, 1000), 24, 8), ((5, 3001), 7, 3), ((2, 3, 640), 0, 0), ((4, 5, 6, 72), 8, 0), ((33,), 0, 1),
                                              ((3, 20000), 5, 1)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_addresses_and_dimensions(shape, gap, offset, dtype):
    say("layer_norm strides", shape, gap, offset, dtype)
    x = rows_of(shape, dtype, 11, gap, offset) if len(shape) > 1 else rows_of((1, *shape), dtype, 11, gap, offset)[0]
    y, mean, rstd, q, s = check_forward(x, *params_of(shape[-1], F32, 12), keep=I8)
    dy = rows_of((int(np.prod(shape[:-1])), shape[-1]), dtype, 13, gap + 1, offset + 1).reshape(x.shape)
    check_backward(dy, x, mean, rstd, *params_of(shape[-1], F32, 12)[:1])


@pytest.mark.parametrize("cols", [100, 2048, 7168, 20000])
def test_values_that_cancel(cols):
    """Rows far off centre, constant rows, rows of zeros, one channel far above the others."""
    say("layer_norm values", cols)
    x = rows_of((8, cols), F32, 14)
    x[0] += 1e4
    x[1] = 7.25
    x[2] = 0
    x[3, cols // 2] = 3e4
    x[4] *= 1e-18
    x[5] *= 1e15
    check_forward(x, *params_of(cols, F32, 15))
    y, _, rstd = Q.layer_norm(x, None, None, EPS)
    assert (y[2] == 0).all() and torch.isfinite(y).all()
    # constant rows and zero eps: 0 times infinity, as the formula has it
    assert torch.isnan(Q.layer_norm(x, None, None, 0.0)[0][2]).all()


@pytest.mark.parametrize("cols", [72, 1024, 7168, 17000])
@pytest.mark.parametrize("keep", [I8, F8])
def test_infinities_and_nans_stay_in_their_rows(cols, keep):
    say("layer_norm special values", cols, keep)
    x = rows_of((6, cols), BF16, 16)
    clean = Q.layer_norm(x, *params_of(cols, F32, 17), keep=keep)
    x[1, cols // 3] = float("nan")
    x[4, cols - 1] = float("inf")
    out = Q.layer_norm(x, *params_of(cols, F32, 17), keep=keep)
    bad = torch.tensor([False, True, False, False, True, False])
    for got, was in zip(out, clean):
        got, was = R.f64(got), R.f64(was)
        assert np.array_equal(got[~bad], was[~bad])
    assert torch.isnan(out[0][bad]).all() and torch.isnan(out[1][1]).all() and torch.isnan(out[4][bad]).all()
    back = Q.restore(out[3], out[4])
    assert torch.isnan(back[bad]).all() and torch.isfinite(back[~bad]).all()


def test_no_rows():
    say("layer_norm no rows")
    w, b = params_of(256, F32, 18)
    x = torch.empty(0, 256, dtype=BF16, device="cuda")
    y, mean, rstd, q, s = Q.layer_norm(x, w, b, keep=I8)
    assert y.shape == (0, 256) and mean.shape == (0,) and q.shape == (0, 256) and s.shape == (0, 2)
    dx, dw, db = Q.layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, 256) and (dw == 0).all() and (db == 0).all()


# ---- backward
def check_backward(dy, x, mean, rstd, w=None, scales=None, out_dtype=None, bias=True):
    dx, dw, db = Q.layer_norm_backward(dy, x, mean, rstd, w, scales=scales, out_dtype=out_dtype, bias=bias)
    cols = dy.shape[-1]
    r = R.f64(rstd).reshape(-1, 1)
    if scales is None:
        away = R.f64(x).reshape(-1, cols) - R.f64(mean).reshape(-1, 1)
        xhat = away * r
        e_xhat = 2 * R.U * np.abs(xhat)
    else:
        xhat = R.values(x, scales)
        e_xhat = R.U * np.abs(xhat)
    ref, bound = R.norm_gradients(R.f64(dy).reshape(-1, cols), xhat, e_xhat, r, None if w is None else R.f64(w))
    assert dx.dtype == (out_dtype or dy.dtype) and dx.shape == dy.shape
    R.check(dx, ref[0], R.stored(bound[0], ref[0], dx.dtype), "dx")
    if w is None:
        assert dw is None and db is None
        return
    assert dw.dtype == w.dtype
    R.check(dw, ref[1], R.stored(bound[1], ref[1], w.dtype), "dweight")
    if bias:
        R.check(db, ref[2], R.stored(bound[2], ref[2], w.dtype), "dbias")
    else:
        assert db is None


def case(rows, cols, dtype, params, keep, seed):
    x = rows_of((rows, cols), dtype, seed)
    w, b = params_of(cols, params, seed + 1)
    out = Q.layer_norm(x, w, b, EPS, keep=keep)
    dy = rows_of((rows, cols), dtype, seed + 2, mean=0.1)
    dy[rows - rows // 8:] = 0
    return (dy, x, out[1], out[2], w) if keep is None else (dy, out[3], None, out[2], w, out[4])


@pytest.mark.parametrize("rows,cols", SIZES + [(4000, 128), (1999, 520), (1300, 3001)])
@pytest.mark.parametrize("dtype,params,keep", [(BF16, F32, None), (BF16, BF16, I8), (F16, F32, F8), (F32, F32, None), (F32, F16, I8), (F16, F16, None)])
def test_backward(rows, cols, dtype, params, keep):
    say("layer_norm_backward", rows, cols, dtype, params, keep)
    check_backward(*case(rows, cols, dtype, params, keep, rows + cols))


@pytest.mark.parametrize("cols", [128, 1000, 4096])
@pytest.mark.parametrize("dy_dtype,x_dtype,out_dtype", [(F32, BF16, BF16), (BF16, F32, F32), (F32, I8, F16), (BF16, F16, None)])
def test_backward_types(cols, dy_dtype, x_dtype, out_dtype):
    say("layer_norm_backward types", cols, dy_dtype, x_dtype, out_dtype)
    keep = x_dtype if x_dtype in (I8, F8) else None
    _, x, mean, rstd, w, *s = case(60, cols, BF16 if keep else x_dtype, F32, keep, 21)
    check_backward(rows_of((60, cols), dy_dtype, 22), x, mean, rstd, w, *s, out_dtype=out_dtype)
    check_backward(rows_of((60, cols), dy_dtype, 22), x, mean, rstd, None, *s)
    check_backward(rows_of((60, cols), dy_dtype, 22), x, mean, rstd, w, *s, bias=False)


def test_backward_of_scales_that_are_no_powers_of_two():
    say("layer_norm_backward quantize scales")
    x = rows_of((50, 900), F32, 23)
    y, mean, rstd = Q.layer_norm(x)
    q, s = Q.quantize(y, I8, Q.QUANT_BLOCK_1x128)
    check_backward(rows_of((50, 900), BF16, 24), q, None, rstd, params_of(900, F32, 25)[0], s)


@pytest.mark.parametrize("cols", [5, 130])
def test_gradients_against_differences(cols):
    """d/dx, d/dw and d/db of sum(y r), from central differences of the formula in 64 bits (step h: error of the order h^2)."""
    say("layer_norm differences", cols)
    rows, h = 4, 1e-5
    x, (w, b), r = rows_of((rows, cols), F32, 26), params_of(cols, F32, 27), rows_of((rows, cols), F32, 28)
    _, mean, rstd = Q.layer_norm(x, w, b, EPS)
    dx, dw, db = Q.layer_norm_backward(r, x, mean, rstd, w)
    x64, w64, b64, r64 = (R.f64(t) for t in (x, w, b, r))
    loss = lambda x, w, b: float((R.norm(x, w, b, EPS)[0][0] * r64).sum())  # noqa: E731

    def differences(i):
        args = [x64, w64, b64]
        g = np.zeros_like(args[i])
        for at in np.ndindex(g.shape):
            up, down = args[i].copy(), args[i].copy()
            up[at] += h
            down[at] -= h
            g[at] = (loss(*args[:i], up, *args[i + 1:]) - loss(*args[:i], down, *args[i + 1:])) / (2 * h)
        return g

    for got, i in ((dx, 0), (dw, 1), (db, 2)):
        ref = differences(i)
        assert np.allclose(R.f64(got), ref, rtol=1e-4, atol=1e-4 * np.abs(ref).max())


@pytest.mark.parametrize("rows,cols", [(3000, 128), (700, 4096), (5, 20000)])
def test_the_same_bits_again_and_on_another_stream(rows, cols):
    say("layer_norm again", rows, cols)
    args = case(rows, cols, BF16, F32, None, 31)
    first = Q.layer_norm_backward(*args)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = Q.layer_norm_backward(*args)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_a_captured_pass():
    say("layer_norm captured")
    x, (w, b), dy = rows_of((500, 1024), BF16, 33), params_of(1024, F32, 34), rows_of((500, 1024), BF16, 35)

    def both():
        y, mean, rstd, q, s = Q.layer_norm(x, w, b, EPS, keep=I8)
        return (y, *Q.layer_norm_backward(dy, q, None, rstd, w, scales=s))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in (36, 37, 38):
        x.copy_(rows_of((500, 1024), BF16, seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, c) for a, c in zip(got, both()))


def test_through_ctypes(monkeypatch):
    say("layer_norm ctypes")
    args = case(37, 1000, BF16, F32, I8, 39)
    x, (w, b) = rows_of((2, 9, 1000), BF16, 40), params_of(1000, BF16, 41)
    want = (*Q.layer_norm(x, w, b, keep=F8), *Q.layer_norm_backward(*args))
    monkeypatch.setattr(Q.ops, "_native_module", False)
    got = (*Q.layer_norm(x, w, b, keep=F8), *Q.layer_norm_backward(*args))
    assert all(np.array_equal(R.f64(a), R.f64(c)) for a, c in zip(want, got))


def test_offsets_beyond_32_bits():
    """Rows whose offsets pass 2^32 elements: the last ones are right."""
    say("layer_norm offsets")
    rows, cols = (1 << 20) + 3, 4160
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    tail = rows_of((5, cols), BF16, 42)
    x[-5:] = tail
    w, b = params_of(cols, F32, 43)
    y, mean, rstd, q, s = Q.layer_norm(x, w, b, keep=I8)
    (ry, rm, rr, rx), (ey, em, er, ex) = R.norm(R.f64(tail), R.f64(w), R.f64(b), EPS)
    R.check(y[-5:], ry, R.stored(ey, ry, BF16), "y")
    R.check(mean[-5:], rm, em + R.U * np.abs(rm), "mean")
    R.check(rstd[-5:], rr, er, "rstd")
    R.check(torch.from_numpy(R.values(q[-5:], s[-5:])), rx, np.repeat(R.f64(s[-5:]), 128, 1)[:, :cols] / 2 + 2 * ex, "kept")
    want = (None, None, rstd[-5:].clone(), q[-5:].clone(), s[-5:].clone())
    del y
    dy = x
    dx, dw, db = Q.layer_norm_backward(dy, q, None, rstd, w, scales=s)
    tx, tw, tb = Q.layer_norm_backward(tail, want[3], None, want[2], w, scales=want[4])
    assert torch.equal(dx[-5:], tx) and torch.allclose(dw, tw, rtol=1e-6, atol=1e-6) and torch.allclose(db, tb, rtol=1e-6, atol=1e-6)
