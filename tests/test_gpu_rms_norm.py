"""Root-mean-square norm, forward and backward, against the formulas in 64 bits, at the sizes, strides and values where it can go wrong."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import language_ref as L
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, F8 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
LARGEST = {I8: 127.0, F8: 448.0}
NAMES = {I8: "int8", F8: "fp8"}


def rows_of(shape, dtype, seed, gap=0, offset=0):
    """Values with channels of different size, in rows `gap` elements longer than they need be."""
    g = torch.Generator().manual_seed(seed)
    rows, cols = int(np.prod(shape[:-1])), shape[-1]
    v = torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g))
    room = torch.full((offset + rows * (cols + gap) + 16,), float("nan"), dtype=dtype, device="cuda")
    t = room[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
    t.copy_(v.to(dtype))
    return t if len(shape) == 2 else t.view(shape) if gap == 0 else t.unflatten(0, shape[:-1])


def weight_of(cols, dtype, seed):
    return (1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def check_forward(x, w, eps=L.EPS, residual=None, out_dtype=None, codes=None, store_y=True):
    out = Q.rms_norm(x, w, eps, residual, out_dtype, codes, store_y)
    y, h, rstd = out[:3]
    cols = x.shape[-1]
    if residual is None:
        assert h is x
    else:
        want = R.f64(x).reshape(-1, cols) + R.f64(residual).reshape(-1, cols)
        assert h.dtype == residual.dtype and h.shape == x.shape
        R.check(h, want, R.stored(R.U * np.abs(want), want, h.dtype), "h")
    (ry, rr), (ey, er) = L.rms(R.f64(h).reshape(-1, cols), None if w is None else R.f64(w), eps)
    assert rstd.shape == x.shape[:-1] and rstd.dtype == F32
    R.check(rstd, rr, er, "rstd")
    if store_y:
        assert y.shape == x.shape and y.dtype == (out_dtype or x.dtype)
        R.check(y, ry, R.stored(ey, ry, y.dtype), "y")
    else:
        assert y is None
    if codes is not None:
        q, s = out[3:]
        assert q.dtype == codes and q.shape == x.shape and s.shape == (*x.shape[:-1], -(-cols // 128))
        L.check_codes(R.f64(q).reshape(-1, cols), R.f64(s).reshape(ry.shape[0], -1), ry, ey, LARGEST[codes], NAMES[codes])
    return out


SIZES = [(1, 1), (3, 5), (2, 8), (5, 64), (300, 64), (17, 127), (513, 128), (9, 130), (100, 257), (33, 512), (5, 1000), (3, 1024), (64, 2048), (7, 2056),
         (1100, 2048), (5, 3001), (3, 4104), (2, 7168), (1200, 7168), (3, 8200), (2, 16384), (2, 16392), (1, 20001), (2, 40000)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype,params,residual,codes", [(BF16, F32, BF16, I8), (F16, F16, None, F8), (F32, F32, F32, None), (BF16, BF16, F32, F8), (F32, BF16, BF16, I8)])
def test_forward(rows, cols, dtype, params, residual, codes):
    say("rms_norm", rows, cols, dtype, params, residual, codes)
    r = None if residual is None else rows_of((rows, cols), residual, rows + cols + 1)
    check_forward(rows_of((rows, cols), dtype, rows + cols), weight_of(cols, params, 3), residual=r, codes=codes)


@pytest.mark.parametrize("rows,cols", [(1, 7168), (300, 128), (40, 1001), (2000, 4096), (3, 20001)])
@pytest.mark.parametrize("codes", [I8, F8])
def test_codes_are_those_of_the_quantiser(rows, cols, codes):
    say("rms_norm codes", rows, cols, codes)
    x, r, w = rows_of((rows, cols), BF16, 4), rows_of((rows, cols), BF16, 5), weight_of(cols, F32, 6)
    x[0] = 0
    r[0] = 0
    y, h, rstd, q, s = Q.rms_norm(x, w, L.EPS, r, F32, codes)
    q2, s2 = Q.quantize(y, codes, Q.QUANT_BLOCK_1x128)
    assert torch.equal(s, s2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
    only = Q.rms_norm(x, w, L.EPS, r, codes=codes, store_y=False)
    assert only[0] is None and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(only[1:], (h, rstd, q, s)))


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [96, 1001, 5000])
def test_forward_without_weight_into_another_type(cols, out_dtype):
    say("rms_norm out_dtype", cols, out_dtype)
    check_forward(rows_of((9, cols), F16, 8), None, out_dtype=out_dtype)


@pytest.mark.parametrize("shape,gap,offset", [((7, 128), 3, 1), ((70, 1000), 24, 8), ((5, 3001), 7, 3), ((2, 3, 640), 0, 0), ((4, 5, 6, 72), 8, 0), ((33,), 0, 1),
                                              ((3, 20000), 5, 1)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_addresses_and_dimensions(shape, gap, offset, dtype):
    say("rms_norm strides", shape, gap, offset, dtype)
    many = shape if len(shape) > 1 else (1, *shape)
    x, r, dy, dh = (rows_of(many, dtype, 11 + i, gap + i, offset + i) for i in range(4))
    if len(shape) == 1:
        x, r, dy, dh = x[0], r[0], dy[0], dh[0]
    w = weight_of(shape[-1], F32, 15)
    _, h, rstd, _, _ = check_forward(x, w, residual=r, codes=I8)
    check_backward(dy, h, rstd, w, dh)


@pytest.mark.parametrize("cols", [100, 2048, 7168, 20000])
def test_values_of_many_sizes(cols):
    """Rows of zeros, one channel far above the others, small and large rows."""
    say("rms_norm values", cols)
    x = rows_of((6, cols), F32, 16)
    x[0] = 0
    x[1, cols // 2] = 3e4
    x[2] *= 1e-18
    x[3] *= 1e15
    x[4, 1:] = 0
    check_forward(x, weight_of(cols, F32, 17), codes=F8)
    assert torch.isnan(Q.rms_norm(x, None, 0.0)[0][0]).all()         # 0 times infinity, as the formula has it


@pytest.mark.parametrize("cols", [72, 1024, 7168, 17000])
@pytest.mark.parametrize("codes", [I8, F8])
def test_infinities_and_nans_stay_in_their_rows(cols, codes):
    say("rms_norm special values", cols, codes)
    x, r, w = rows_of((6, cols), BF16, 18), rows_of((6, cols), BF16, 19), weight_of(cols, F32, 20)
    clean = Q.rms_norm(x, w, L.EPS, r, codes=codes)
    x[1, cols // 3] = float("nan")
    r[4, cols - 1] = float("inf")
    out = Q.rms_norm(x, w, L.EPS, r, codes=codes)
    bad = torch.tensor([False, True, False, False, True, False])
    for got, was in zip(out, clean):
        assert np.array_equal(R.f64(got)[~bad], R.f64(was)[~bad])
    assert torch.isnan(out[0][1]).all() and torch.isnan(out[0][4, cols - 1]) and out[2][4] == 0
    assert torch.isnan(out[4][1]).all() and torch.isnan(out[4][4, -1])
    assert torch.isnan(Q.restore(out[3], out[4])[1]).all()


def test_no_rows():
    say("rms_norm no rows")
    w, x = weight_of(256, F32, 21), torch.empty(0, 256, dtype=BF16, device="cuda")
    y, h, rstd, q, s = Q.rms_norm(x, w, residual=x, codes=I8)
    assert y.shape == h.shape == q.shape == (0, 256) and rstd.shape == (0,) and s.shape == (0, 2)
    dx, dw = Q.rms_norm_backward(x, h, rstd, w)
    assert dx.shape == (0, 256) and (dw == 0).all()


# ---- backward
def check_backward(dy, h, rstd, w=None, dh=None, out_dtype=None):
    dx, dw = Q.rms_norm_backward(dy, h, rstd, w, dh, out_dtype)
    cols = dy.shape[-1]
    flat = lambda t: None if t is None else R.f64(t).reshape(-1, cols)  # noqa: E731
    (rx, rw), (ex, ew) = L.rms_gradients(flat(dy), flat(h), R.f64(rstd).reshape(-1, 1), None if w is None else R.f64(w), flat(dh))
    assert dx.dtype == (out_dtype or dy.dtype) and dx.shape == dy.shape
    R.check(dx, rx, R.stored(ex, rx, dx.dtype), "dx")
    if w is None:
        assert dw is None
    else:
        assert dw.dtype == w.dtype and dw.shape == w.shape
        R.check(dw, rw, R.stored(ew, rw, w.dtype), "dw")
    return dx, dw


def gradients_case(rows, cols, dtype, params, residual, seed):
    h, w = rows_of((rows, cols), dtype, seed), weight_of(cols, params, seed + 1)
    rstd = Q.rms_norm(h, w)[2]
    return rows_of((rows, cols), dtype, seed + 2), h, rstd, w, rows_of((rows, cols), dtype, seed + 3) if residual else None


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype,params,residual", [(BF16, F32, True), (F16, F16, False), (F32, F32, True), (BF16, BF16, True)])
def test_backward(rows, cols, dtype, params, residual):
    say("rms_norm_backward", rows, cols, dtype, params, residual)
    check_backward(*gradients_case(rows, cols, dtype, params, residual, rows + cols))


@pytest.mark.parametrize("cols", [72, 1001, 7168, 17000])
@pytest.mark.parametrize("dy_dtype,h_dtype,dh_dtype,out_dtype", [(F32, BF16, F16, BF16), (BF16, F32, F32, F32), (F16, BF16, BF16, F32), (F32, F32, BF16, F16)])
def test_backward_types(cols, dy_dtype, h_dtype, dh_dtype, out_dtype):
    say("rms_norm_backward types", cols, dy_dtype, h_dtype, dh_dtype, out_dtype)
    h = rows_of((19, cols), h_dtype, 31)
    check_backward(rows_of((19, cols), dy_dtype, 32), h, Q.rms_norm(h)[2], weight_of(cols, BF16, 33), rows_of((19, cols), dh_dtype, 34), out_dtype)
    check_backward(rows_of((19, cols), dy_dtype, 32), h, Q.rms_norm(h)[2], None, None, out_dtype)


@pytest.mark.parametrize("cols", [40, 1000])
def test_backward_against_differences(cols):
    """Central differences in 64 bits of sum(y r) + sum(h t) along 8 directions."""
    say("rms_norm differences", cols)
    x, res, w = rows_of((6, cols), F32, 35), rows_of((6, cols), F32, 36), weight_of(cols, F32, 37)
    r, t = rows_of((6, cols), F32, 38), rows_of((6, cols), F32, 39)
    _, h, rstd = Q.rms_norm(x, w, L.EPS, res)
    dx, dw = Q.rms_norm_backward(r, h, rstd, w, dh=t)
    X, W, RR, T = (R.f64(v) for v in (h, w, r, t))

    def value(X, W):
        return (L.rms(X, W, L.EPS)[0][0] * RR).sum() + (X * T).sum()

    rng = np.random.default_rng(1)
    for _ in range(8):
        a, b, step = rng.standard_normal(X.shape), rng.standard_normal(W.shape), 1e-5
        got = (R.f64(dx) * a).sum() + (R.f64(dw) * b).sum()
        want = (value(X + step * a, W + step * b) - value(X - step * a, W - step * b)) / (2 * step)
        size = np.sqrt((R.f64(dx) ** 2).sum() + (R.f64(dw) ** 2).sum())
        assert abs(got - want) <= 1e-4 * size


@pytest.mark.parametrize("rows,cols", [(3000, 128), (700, 4096), (5, 20000)])
def test_the_same_bits_again_and_on_another_stream(rows, cols):
    say("rms_norm again", rows, cols)
    args = gradients_case(rows, cols, BF16, F32, True, 41)
    first = Q.rms_norm_backward(*args)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = Q.rms_norm_backward(*args)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_a_captured_pass():
    say("rms_norm captured")
    x, r, dy = (rows_of((500, 1024), BF16, 43 + i) for i in range(3))
    w = weight_of(1024, F32, 46)

    def both():
        y, h, rstd, q, s = Q.rms_norm(x, w, L.EPS, r, codes=I8)
        return (y, h, q, s, *Q.rms_norm_backward(dy, h, rstd, w, dh=y))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in (47, 48, 49):
        x.copy_(rows_of((500, 1024), BF16, seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, c) for a, c in zip(got, both()))


def test_through_ctypes(monkeypatch):
    say("rms_norm ctypes")
    args = gradients_case(37, 1000, BF16, F32, True, 51)
    x, r, w = rows_of((2, 9, 1000), BF16, 52), rows_of((2, 9, 1000), F32, 53), weight_of(1000, BF16, 54)
    want = (*Q.rms_norm(x, w, residual=r, codes=F8), *Q.rms_norm_backward(*args))
    monkeypatch.setattr(Q.ops, "_native_module", False)
    got = (*Q.rms_norm(x, w, residual=r, codes=F8), *Q.rms_norm_backward(*args))
    assert all(np.array_equal(R.f64(a), R.f64(c)) for a, c in zip(want, got))


def test_offsets_beyond_32_bits():
    """Rows whose offsets pass 2^32 elements: the last ones are right."""
    say("rms_norm offsets")
    rows, cols = (1 << 20) + 3, 4160
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    tail, w = rows_of((5, cols), BF16, 55), weight_of(cols, F32, 56)
    x[-5:] = tail
    y, h, rstd, q, s = Q.rms_norm(x, w, codes=I8)
    want = Q.rms_norm(tail, w, codes=I8)
    assert all(torch.equal(a[-5:], b) for a, b in zip((y, rstd, q, s), (want[0], *want[2:])))
    del y, q
    dx, dw = Q.rms_norm_backward(x, x, rstd, w, dh=x)
    tx, tw = Q.rms_norm_backward(tail, tail, want[2], w, dh=tail)
    assert torch.equal(dx[-5:], tx) and torch.allclose(dw, tw, rtol=1e-6, atol=1e-6)
