"""The norm's 8-bit codes bit for bit: scales are the fp32 quotients max|y| / 448 (127), rounded to nearest, and codes the fp32 quotients y / s, rounded to nearest even; none a step
away because a quotient was taken for a product with a reciprocal."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests.util import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes,largest", [(torch.float8_e4m3fn, 448), (torch.int8, 127)])
@pytest.mark.parametrize("rows,cols", [(1, 7168), (300, 1001), (40, 20000)])
@pytest.mark.parametrize("seed", range(5))
def test_codes_and_scales_are_rounded_quotients(rows, cols, codes, largest, seed):
    say("norm codes", rows, cols, codes, seed)
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g))).bfloat16().cuda()
    r, w = (2 * torch.randn(rows, cols, generator=g)).bfloat16().cuda(), (1 + 0.2 * torch.randn(cols, generator=g)).bfloat16().cuda()
    y, _, _, q, s = Q.rms_norm(x, w, 1e-6, residual=r, out_dtype=torch.float32, codes=codes)
    y = np.pad(y.cpu().numpy(), ((0, 0), (0, -cols % 128))).reshape(rows, -1, 128)
    scale = np.abs(y).max(-1, keepdims=True) / np.float32(largest)
    assert scale.dtype == np.float32 and np.array_equal(s.cpu().numpy(), scale[..., 0])
    v = torch.from_numpy((y / scale).reshape(rows, -1)[:, :cols].copy())
    want = v.to(codes).float() if codes != torch.int8 else torch.round(v)
    assert torch.equal(q.cpu().float(), want)
    only = Q.rms_norm(x, w, 1e-6, residual=r, codes=codes, store_y=False)
    assert torch.equal(only[3].view(torch.uint8), q.view(torch.uint8)) and torch.equal(only[4], s)
