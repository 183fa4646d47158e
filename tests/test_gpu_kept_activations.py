"""Activations in 8 bits under powers of two, and back: bit for bit against their definition."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, F8 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


def check_exact(x, dtype):
    cols = x.shape[-1]
    q, s = Q.checkpoint(x, dtype)
    assert q.shape == x.shape and s.shape == (*x.shape[:-1], -(-cols // 128))
    x64 = R.f64(x).reshape(-1, cols)
    scales = R.scales_of(x64, dtype)
    assert np.array_equal(R.f64(s).reshape(scales.shape), scales)
    codes = R.codes_of(x64, scales, dtype)
    assert np.array_equal(R.f64(q).reshape(-1, cols), codes)
    for out in (F32, BF16):
        back = Q.restore(q, s, out)
        assert back.shape == x.shape and back.dtype == out
        assert np.array_equal(R.f64(back).reshape(-1, cols), R.values(q, s))          # exact in both
    return q, s


@pytest.mark.parametrize("rows,cols", [(1, 1), (4, 3), (1, 8), (7, 100), (5, 128), (33, 129), (16, 2048), (3, 2049), (200, 1000), (2, 14336), (70000, 24)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("codes", [I8, F8])
def test_round_trip(rows, cols, dtype, codes):
    say("checkpoint", rows, cols, dtype, codes)
    g = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    check_exact(x.to(dtype).cuda(), codes)


@pytest.mark.parametrize("codes", [I8, F8])
def test_edges_of_a_scale(codes):
    """Maxima at, just below and just above the largest code under a power of two; ties; zeros; the smallest numbers."""
    say("checkpoint edges", codes)
    top = R.LARGEST[codes]
    x = torch.zeros(12, 256)
    for i, v in enumerate((top, np.nextafter(np.float32(top), np.float32(0)), np.nextafter(np.float32(top), np.float32(1e9)), 2 * top, top / 1024)):
        x[i] = torch.linspace(-1, 1, 256)
        x[i, 17] = float(v)
        x[i, 200] = -float(v)
    x[5, :128] = torch.arange(128) + 0.5
    x[5, 0] = top
    x[6, 3] = 2.0 ** -126
    x[7, 3] = -2.0 ** -149
    x[8] = torch.linspace(-top, top, 256)
    x[9] = torch.exp2(torch.linspace(-20, 8, 256))
    check_exact(x.cuda(), codes)
    assert (Q.checkpoint(torch.zeros(2, 130, device="cuda"), codes)[1] == 1).all()


@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_the_largest_numbers_stay_finite(dtype, codes):
    say("checkpoint largest", dtype, codes)
    big = torch.finfo(dtype).max
    x = torch.tensor([[big, -big, big / 2, 1.0, big * 0.98]], dtype=dtype, device="cuda")
    back = Q.restore(*Q.checkpoint(x, codes), dtype)
    assert torch.isfinite(back).all()
    assert torch.allclose(back[0, :3].double(), x[0, :3].double(), rtol=0.07)


@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_anything_else_reads_as_nan(codes, bad):
    say("checkpoint special", codes, bad)
    x = torch.randn(3, 400, generator=torch.Generator().manual_seed(1)).cuda()
    want = Q.restore(*Q.checkpoint(x, codes), F32)
    x[1, 130] = bad
    q, s = Q.checkpoint(x, codes)
    back = Q.restore(q, s, F32)
    assert torch.isnan(back[1, 128:256]).all()
    keep = torch.ones_like(back, dtype=torch.bool)
    keep[1, 128:256] = False
    assert torch.equal(back[keep], want[keep])


@pytest.mark.parametrize("gap,offset", [(3, 1), (8, 0), (1, 7)])
@pytest.mark.parametrize("cols", [5, 300, 2051])
def test_strides_and_addresses(cols, gap, offset):
    say("checkpoint strides", cols, gap, offset)
    room = torch.full((offset + 20 * (cols + gap),), float("nan"), dtype=BF16, device="cuda")
    x = room[offset:].view(20, cols + gap)[:, :cols]
    x.copy_(torch.randn(20, cols, generator=torch.Generator().manual_seed(cols)))
    q, s = check_exact(x, I8)
    wide = torch.zeros(20, cols + gap, dtype=I8, device="cuda")
    wide[:, :cols] = q
    assert torch.equal(Q.restore(wide[:, :cols], s), Q.restore(q, s))
    assert torch.equal(Q.restore(q.view(4, 5, cols), s.view(4, 5, -1)).view(20, cols), Q.restore(q, s))


def test_codes_of_the_quantiser():
    say("restore quantize")
    x = torch.randn(40, 900, generator=torch.Generator().manual_seed(2)).cuda()
    for codes in (I8, F8):
        q, s = Q.quantize(x, codes, Q.QUANT_BLOCK_1x128)
        assert np.array_equal(R.f64(Q.restore(q, s, F32)), R.values(q, s).astype(np.float32))


def test_no_rows_and_ctypes(monkeypatch):
    say("checkpoint no rows")
    x = torch.randn(9, 333, generator=torch.Generator().manual_seed(3)).to(F16).cuda()
    q, s = Q.checkpoint(x, F8)
    empty = Q.checkpoint(x[:0], I8)
    assert empty[0].shape == (0, 333) and Q.restore(*empty).shape == (0, 333)
    monkeypatch.setattr(Q.ops, "_native_module", False)
    q2, s2 = Q.checkpoint(x, F8)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    assert torch.equal(Q.restore(q, s, F16), Q.restore(q2, s2, F16))


def test_offsets_beyond_32_bits():
    say("checkpoint offsets")
    rows, cols = 70000, 65536
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    tail = torch.randn(2, cols, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    x[-2:] = tail
    q, s = Q.checkpoint(x, I8)
    tq, ts = Q.checkpoint(tail, I8)
    assert torch.equal(q[-2:], tq) and torch.equal(s[-2:], ts)
    del x
    assert torch.equal(Q.restore(q, s)[-2:], Q.restore(tq, ts))
