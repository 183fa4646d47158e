"""What a code times its scale is in 16 bits: exact where that can be, one rounding of the fp32 product where not."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, F8 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


def every_code(codes):
    """All finite codes of a type, 128 to a block, on the host."""
    q = torch.arange(-127, 128, dtype=torch.int16).to(torch.int8) if codes == I8 else None
    if codes == F8:
        bits = torch.arange(256, dtype=torch.int16).to(torch.uint8)
        q = bits[(bits & 0x7F) != 0x7F].view(F8)
    return q


def under(q, scales):
    """[scales, codes] codes and their blocks' scales."""
    n, blocks = q.shape[0], -(-q.shape[0] // 128)
    many = q.view(torch.uint8).repeat(len(scales), 1).view(q.dtype)
    return many, torch.tensor(scales, dtype=F32)[:, None].repeat(1, blocks)


@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("out", [BF16, F16, F32])
def test_restore_rounds_the_product_of_fp32(codes, out):
    say("restore rounds", codes, out)
    q, s = under(every_code(codes), [2.0 ** e for e in (-126, -125, -124, -120, -60, -30, -24, -20, -14, 0, 5, 9)] + [1 / 3, 0.37, 3.3e-5, 1.7e-38, 4.7e-7])
    want = (q.float() * s.repeat_interleave(128, 1)[:, :q.shape[1]]).to(out)
    assert torch.equal(Q.restore(q.cuda(), s.cuda(), out).cpu(), want)


@pytest.mark.parametrize("codes,out,least,beyond", [(I8, BF16, -126, None), (F8, BF16, -124, -126), (I8, F16, -24, -25), (F8, F16, -15, -16)])
def test_where_a_power_of_two_is_exact(codes, out, least, beyond):
    """From the smallest scale on whose codes are multiples of the type's smallest number; half of that number off below."""
    say("restore exact", codes, out, least)
    code = every_code(codes)
    exact = lambda e: R.f64(code)[None] * 2.0 ** e  # noqa: E731
    back = lambda e: R.f64(Q.restore(*(t.cuda() for t in under(code, [2.0 ** e])), out))  # noqa: E731
    assert np.array_equal(back(least), exact(least)) and np.array_equal(back(5), exact(5))
    if beyond is not None:
        off = np.abs(back(beyond) - exact(beyond))
        assert 0 < off.max() <= R.LEAST[out]


@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("dtype,scale", [(F16, 2.0 ** -26), (F16, 2.0 ** -17), (BF16, 2.0 ** -40), (BF16, 0.37)])
def test_weight_gradient_of_small_values(codes, dtype, scale):
    """v is q s in dy's type, its smallest numbers included: the product is that of these values."""
    say("weight_gradient small values", codes, dtype, scale)
    g = torch.Generator().manual_seed(3)
    dy = torch.randn(100, 70, generator=g).to(dtype)
    code = every_code(codes).view(torch.uint8)
    q = code[torch.randint(0, len(code), (100, 300), generator=g)].view(codes)
    s = torch.full((100, 3), scale)
    v = (q.float() * scale).to(dtype)
    ref, bound = R.weight_gradient(R.f64(dy), R.f64(v), None, None)
    dw, _ = Q.weight_gradient(dy.cuda(), q.cuda(), s.cuda())
    R.check(dw, ref[0], bound[0] + R.U * np.abs(ref[0]), "dw")
