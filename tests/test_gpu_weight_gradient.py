"""The weight gradient out of activations in 8 bits, against the formula in 64 bits."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, F8 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


def operands(rows, n, cols, dtype, codes, norm, seed):
    g = torch.Generator().manual_seed(seed)
    dy = (torch.randn(rows, n, generator=g) * n ** -0.5).to(dtype).cuda()
    x = (torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g))).cuda()
    q, s = Q.checkpoint(x, codes)
    w = b = None
    if norm:
        w, b = (1 + 0.2 * torch.randn(cols, generator=g)).to(dtype).cuda(), (0.1 * torch.randn(cols, generator=g)).to(dtype).cuda()
    return dy, q, s, w, b


def check(dy, q, s, w=None, b=None, out=F32, got=None):
    dw, db = got or Q.weight_gradient(dy, q, s, w, b, out_dtype=out)
    n, cols = dy.shape[-1], q.shape[-1]
    assert dw.shape == (n, cols) and dw.dtype == out and db.shape == (n,) and db.dtype == F32
    v = R.values(q, s)
    ref, bound = R.weight_gradient(R.f64(dy).reshape(-1, n), v, None if w is None else R.f64(w), None if b is None else R.f64(b))
    R.check(dw, ref[0], R.stored(bound[0], ref[0], out), "dw")
    R.check(db, ref[1], bound[1] + R.U * np.abs(ref[1]), "db")


@pytest.mark.parametrize("rows,n,cols", [(1, 1, 1), (1, 300, 200), (2, 7, 9), (63, 8, 130), (64, 128, 128), (65, 129, 127), (130, 1, 500), (100, 500, 1),
                                         (200, 256, 512), (513, 260, 1000), (1000, 33, 2000), (999, 1001, 257), (4100, 64, 64), (3000, 520, 3), (640, 1300, 700)])
@pytest.mark.parametrize("dtype,codes,norm,out", [(BF16, I8, True, F32), (F16, F8, False, F32), (BF16, F8, False, BF16), (F16, I8, True, F16)])
def test_sizes(rows, n, cols, dtype, codes, norm, out):
    say("weight_gradient", rows, n, cols, dtype, codes, norm, out)
    check(*operands(rows, n, cols, dtype, codes, norm, rows + n + cols), out=out)


@pytest.mark.parametrize("params", [F32, BF16, F16])
@pytest.mark.parametrize("bias", [False, True])
def test_parameters(params, bias):
    say("weight_gradient parameters", params, bias)
    dy, q, s, w, b = operands(300, 200, 330, BF16, I8, True, 5)
    check(dy, q, s, w.to(params), b.to(params) if bias else None)


@pytest.mark.parametrize("gap_dy,gap_q,offset", [(1, 0, 0), (0, 3, 1), (5, 8, 3), (8, 16, 8)])
@pytest.mark.parametrize("rows,n,cols", [(130, 72, 136), (300, 257, 129), (70, 6, 5)])
def test_strides_and_addresses(rows, n, cols, gap_dy, gap_q, offset):
    say("weight_gradient strides", rows, n, cols, gap_dy, gap_q, offset)
    dy, q, s, w, b = operands(rows, n, cols, BF16, I8, True, 7)

    def within(t, gap, fill):
        room = torch.full((offset + rows * (t.shape[1] + gap),), fill, dtype=t.dtype, device="cuda")
        view = room[offset:].view(rows, t.shape[1] + gap)[:, :t.shape[1]]
        return view.copy_(t)

    want = Q.weight_gradient(dy, q, s, w, b)
    got = Q.weight_gradient(within(dy, gap_dy, float("nan")), within(q, gap_q, 99), s, w, b)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    check(dy, q, s, w, b, got=got)


def test_more_dimensions_and_no_rows():
    say("weight_gradient dimensions")
    dy, q, s, w, b = operands(60, 40, 200, BF16, F8, True, 8)
    want = Q.weight_gradient(dy, q, s, w, b)
    got = Q.weight_gradient(dy.view(3, 20, 40), q.view(3, 20, 200), s.view(3, 20, 2), w, b)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    dw, db = Q.weight_gradient(dy[:0], q[:0], s[:0], w, b)
    assert dw.shape == (40, 200) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("rows,n,cols", [(70, 200, 300), (5000, 128, 128)])
def test_special_values_stay_where_they_belong(rows, n, cols):
    """A NaN of dy makes one row of dw NaN, a block that reads as NaN its columns; a row beyond the last makes none."""
    say("weight_gradient special values", rows, n, cols)
    dy, q, s, _, _ = operands(rows, n, cols, BF16, I8, False, 9)
    clean = Q.weight_gradient(dy, q, s)[0]
    dy[rows - 1, 3] = float("nan")
    dw, db = Q.weight_gradient(dy, q, s)
    assert torch.isnan(dw[3]).all() and torch.isnan(db[3]) and torch.isnan(dw).sum() == cols and torch.isnan(db).sum() == 1
    assert torch.equal(dw[4:], clean[4:])
    s[rows // 2, 0] = float("nan")
    dy[rows - 1, 3] = 0
    dw, _ = Q.weight_gradient(dy, q, s)
    edge = min(cols, 128)
    assert torch.isnan(dw[:, :edge]).all() and torch.isfinite(dw[:, edge:]).all()


@pytest.mark.parametrize("rows,n,cols,config", [(999, 8190, 1021, "256x128"), (2048, 2047, 7168, "256x256"), (4000, 512, 1030, "128x128_split"),
                                                (16384, 1024, 4095, "256x256_split"), (32700, 512, 1020, "256x128_split"), (700, 1024, 1024, "128x128")])
@pytest.mark.parametrize("dtype,codes,norm,out", [(BF16, I8, True, F32), (F16, F8, False, BF16)])
def test_every_tile(rows, n, cols, config, dtype, codes, norm, out):
    """Sizes that the tiles are chosen for, whole and split, against the formula in 64 bits on the GPU."""
    say("weight_gradient tiles", rows, n, cols, dtype, codes, norm, out)
    dy, q, s, w, b = operands(rows, n, cols, dtype, codes, norm, rows + n)
    dw, db = Q.weight_gradient(dy, q, s, w, b, out_dtype=out)
    assert Q.last_config().startswith("weight_gradient_" + config)
    v = q.double() * s.double().repeat_interleave(128, 1)[:, :cols]
    d = dy.double()
    adds = (rows / 4 + 48) * R.U                          # as in training_ref.weight_gradient
    ref, bound = torch.mm(d.t().contiguous(), v), adds * torch.mm(d.t().contiguous().abs(), v.abs())
    sums, e_sums = d.sum(0), adds * d.abs().sum(0)
    assert ((db.double() - sums).abs() <= e_sums + R.U * sums.abs()).all()
    if norm:
        w, b = w.double(), b.double()
        scaled, rank1 = ref * w, sums[:, None] * b
        bound = bound * w.abs() + 2 * R.U * scaled.abs() + e_sums[:, None] * b.abs() + 2 * R.U * ((scaled + rank1).abs() + 2 * rank1.abs())
        ref = scaled + rank1
    bound = bound * (1 + R.HALF_STEP[out]) + R.HALF_STEP[out] * ref.abs() + R.LEAST[out]
    assert ((dw.double() - ref).abs() <= bound).all()


def test_scales_that_are_no_powers_of_two():
    """q s is rounded to dy's type then: half a last place of each value more."""
    say("weight_gradient quantize scales")
    dy, _, _, _, _ = operands(500, 140, 300, F16, I8, False, 10)
    q, s = Q.quantize(torch.randn(500, 300, generator=torch.Generator().manual_seed(11)).cuda(), I8, Q.QUANT_BLOCK_1x128)
    dw, db = Q.weight_gradient(dy, q, s)
    ref, bound = R.weight_gradient(R.f64(dy), R.values(q, s), None, None)
    more = (R.HALF_STEP[F16] * 1.01) * (np.abs(R.f64(dy)).T @ np.abs(R.values(q, s)))
    R.check(dw, ref[0], bound[0] + more, "dw")


@pytest.mark.parametrize("rows,n,cols", [(3000, 256, 256), (777, 1500, 900)])
def test_the_same_bits_again_on_streams_and_captured(rows, n, cols):
    say("weight_gradient again", rows, n, cols)
    args = operands(rows, n, cols, BF16, I8, True, 12)
    want = Q.weight_gradient(*args)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = Q.weight_gradient(*args)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, c) for a, c in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = Q.weight_gradient(*args)
    for seed in (13, 14, 15):
        args[0].copy_(operands(rows, n, cols, BF16, I8, True, seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, c) for a, c in zip(got, Q.weight_gradient(*args)))


def test_through_ctypes(monkeypatch):
    say("weight_gradient ctypes")
    args = operands(200, 100, 300, F16, F8, True, 16)
    want = Q.weight_gradient(*args)
    monkeypatch.setattr(Q.ops, "_native_module", False)
    assert all(torch.equal(a, c) for a, c in zip(want, Q.weight_gradient(*args)))


def test_a_step_of_training():
    """Norm and linear layer together: gradients out of 8 bits against those of the formulas with the same codes."""
    say("training step")
    g = torch.Generator().manual_seed(17)
    rows, cols, n = 700, 512, 384
    x, W, dz = torch.randn(rows, cols, generator=g).cuda(), (torch.randn(n, cols, generator=g) * cols ** -0.5).to(BF16).cuda(), None
    w, b = (1 + 0.2 * torch.randn(cols, generator=g)).cuda(), (0.1 * torch.randn(cols, generator=g)).cuda()
    dz = torch.randn(rows, n, generator=g).to(BF16).cuda()
    _, _, rstd, q, s = Q.layer_norm(x, w, b, keep=I8)
    check(dz, q, s, w, b)
    dy = Q.gemm(dz, W, torch.empty(rows, cols, device="cuda"), "kn")
    dx, dw, db = Q.layer_norm_backward(dy, q, None, rstd, w, scales=s)
    dy64 = R.f64(dz) @ R.f64(W)
    ref, _ = R.norm_gradients(dy64, R.values(q, s), 0 * dy64, R.f64(rstd)[:, None], R.f64(w))
    for got, want in zip((dx, dw, db), ref):
        assert np.linalg.norm(R.f64(got) - want) <= 1e-5 * np.linalg.norm(want)          # fp32 sums of 384 and 700 terms


def test_offsets_beyond_32_bits():
    say("weight_gradient offsets")
    rows, n, cols = 150000, 16384, 32768
    q, s = torch.zeros(rows, cols, dtype=I8, device="cuda"), torch.ones(rows, cols // 128, device="cuda")
    dy = torch.zeros(rows, n, dtype=BF16, device="cuda")
    g = torch.Generator().manual_seed(18)
    dy[-3:] = torch.randn(3, n, generator=g).to(BF16).cuda()
    q[-3:] = torch.randint(-127, 128, (3, cols), generator=g, dtype=I8).cuda()
    dw, db = Q.weight_gradient(dy[:, -64:], q[:, -192:], s[:, -2:].contiguous())
    tw, tb = Q.weight_gradient(dy[-3:, -64:], q[-3:, -192:], s[-3:, -2:].contiguous())
    assert torch.allclose(dw, tw, rtol=1e-6, atol=1e-6) and torch.allclose(db, tb, rtol=1e-6, atol=1e-6)
