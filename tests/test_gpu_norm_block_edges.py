"""Layer norm's backward pass out of codes where the row ends a few columns into a block: the last octet of a row reaches back into the block in
front, which has a scale of its own.  Widths put the octet it shares elements with into the same wave, an earlier pass of it, and another wave."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, F8 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


def operands(rows, cols, codes, dtype, tail, seed):
    """dy, codes and scales of an xhat whose last block is `tail` times the rest, rstd, weight."""
    g = torch.Generator().manual_seed(seed)
    xhat = torch.randn(rows, cols, generator=g)
    xhat[:, cols // 128 * 128:] *= tail
    q, s = Q.checkpoint(xhat.cuda(), codes)
    dy = torch.randn(rows, cols, generator=g).to(dtype).cuda()
    return dy, q, s, (0.5 + torch.rand(rows, generator=g)).cuda(), (1 + 0.2 * torch.randn(cols, generator=g)).cuda()


@pytest.mark.parametrize("cols", [129, 135, 257, 263, 385, 513, 517, 519, 641, 1025, 1031, 1537, 2049, 2055, 4097, 8193, 8199, 16257])
@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("dtype,out,tail", [(F32, F32, 2.0 ** -6), (BF16, F32, 2.0 ** 6), (F16, BF16, 2.0 ** -6)])
def test_a_row_that_ends_behind_the_edge_of_a_block(cols, codes, dtype, out, tail):
    say("layer_norm_backward block edge", cols, codes, dtype, out, tail)
    dy, q, s, rstd, w = operands(37, cols, codes, dtype, tail, cols)
    dx, dw, db = Q.layer_norm_backward(dy, q, None, rstd, w, scales=s, out_dtype=out)
    xhat = R.values(q, s)
    ref, bound = R.norm_gradients(R.f64(dy), xhat, R.U * np.abs(xhat), R.f64(rstd)[:, None], R.f64(w))
    R.check(dx, ref[0], R.stored(bound[0], ref[0], out), "dx")
    R.check(dw, ref[1], R.stored(bound[1], ref[1], F32), "dweight")
    R.check(db, ref[2], R.stored(bound[2], ref[2], F32), "dbias")


@pytest.mark.parametrize("cols", [517, 1025, 4097, 8193])
def test_the_same_bits_again(cols):
    say("layer_norm_backward block edge again", cols)
    dy, q, s, rstd, w = operands(700, cols, I8, BF16, 2.0 ** -6, cols)
    first = Q.layer_norm_backward(dy, q, None, rstd, w, scales=s)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, Q.layer_norm_backward(dy, q, None, rstd, w, scales=s)))
