"""Adapters of many requests at once, forward and backward, against the formulas in 64 bits."""
import numpy as np
import pytest
import torch

import qgemm_amd as Q
from tests import language_ref as L
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def values(shape, dtype, seed, scale=1.0, gap=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    rows, cols = int(np.prod(shape[:-1])), shape[-1]
    v = torch.randn(rows, cols, generator=g) * scale
    room = torch.full((offset + rows * (cols + gap) + 16,), float("nan"), dtype=dtype, device="cuda")
    t = room[offset:offset + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
    t.copy_(v.to(dtype))
    return t if len(shape) == 2 else t.view(shape) if gap == 0 else t.unflatten(0, shape[:-1])


def ids_of(rows, adapters, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "mixed":                                    # in any order, some of none
        ids = torch.randint(-1, adapters, (rows,), generator=g)
    elif kind == "runs":                                   # prompts side by side
        ids = torch.sort(torch.randint(0, adapters, (rows,), generator=g)).values.flip(0)
    elif kind == "one":
        ids = torch.full((rows,), adapters - 1)
    else:                                                  # numbers that name none
        ids = torch.tensor([-1, adapters, -100, 2 ** 31 - 1]).repeat(rows)[:rows]
    return ids


def operands(rows, adapters, rank, k, n, dtype, y_dtype, seed):
    return (values((rows, n), y_dtype, seed), values((rows, k), dtype, seed + 1), values((adapters, rank, k), dtype, seed + 2, k ** -0.5),
            values((adapters, rank, n), dtype, seed + 3, 0.5), 0.5 + torch.rand(adapters, generator=torch.Generator().manual_seed(seed + 4)).cuda())


def check(y, x, A, B, ids, scaling, out=None):
    groups = Q.group_rows(ids.cuda(), len(A))
    was = R.f64(y).reshape(-1, y.shape[-1])
    got, u = Q.add_adapters(y, x, A, B, groups, scaling, out=out, keep=True)
    s = np.ones(len(A)) if scaling is None else R.f64(scaling)
    (ro, ru), (eo, eu) = L.adapters(was, R.f64(x).reshape(-1, x.shape[-1]), R.f64(A), R.f64(B), ids.numpy().reshape(-1), s, 3 if y.dtype == F32 else 2)
    assert got.dtype == y.dtype and got.shape == y.shape and u.dtype == F32 and u.shape == (*x.shape[:-1], A.shape[1])
    R.check(u, ru, eu + R.U * np.abs(ru), "u")
    R.check(got, ro, R.stored(eo, ro, y.dtype), "out")
    again = Q.add_adapters(torch.from_numpy(was).to(y.dtype).cuda().view(y.shape), x, A, B, groups, scaling)
    assert torch.equal(again, got)                         # (without u, in a new tensor)
    return got, u, groups


def check_backward(dy, x, u, A, B, ids, scaling, dx, grad_dtype=F32):
    groups = Q.group_rows(ids.cuda(), len(A))
    got = Q.add_adapters_backward(dy, x, u, A, B, groups, scaling, dx=dx, grad_dtype=grad_dtype)
    s = np.ones(len(A)) if scaling is None else R.f64(scaling)
    k, n = x.shape[-1], dy.shape[-1]
    base = np.zeros((ids.numel(), k)) if dx is None else R.f64(dx).reshape(-1, k)
    dx_dtype = x.dtype if dx is None else dx.dtype
    ref, bound = L.adapter_gradients(R.f64(dy).reshape(-1, n), R.f64(x).reshape(-1, k), R.f64(u).reshape(-1, A.shape[1]), R.f64(A), R.f64(B), ids.numpy().reshape(-1), s, base,
                                     3 if dx_dtype == F32 else 2, 3 if grad_dtype == F32 else 2)
    for g, r, e, t, name in zip(got, ref, bound, (dx_dtype, grad_dtype, grad_dtype), ("dx", "dA", "dB")):
        assert g.dtype == t
        R.check(g, r, R.stored(e, r, t), name)
    assert got[0].shape == x.shape and got[1].shape == A.shape and got[2].shape == B.shape
    return got


@pytest.mark.parametrize("rows,adapters,kind", [(1, 1, "one"), (1, 3, "none"), (5, 40, "mixed"), (64, 48, "mixed"), (200, 3, "runs"), (1000, 7, "mixed"), (129, 2, "none"),
                                                (4097, 300, "mixed"), (3000, 1, "one"), (70, 65535, "mixed"), (0, 5, "mixed"), (16384, 3, "runs"), (16385, 5, "mixed"), (40001, 7, "mixed"), (40000, 2, "runs"), (20000, 30000, "mixed"),
                                                (257, 257, "mixed"), (256, 256, "runs"), (2049, 2048, "mixed"), (2048, 2049, "mixed")])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_groups(rows, adapters, kind, dtype):
    """Rows group by group in their own order, and slots that cover every group in pieces of up to 64."""
    say("group_rows", rows, adapters, kind, dtype)
    ids = ids_of(rows, adapters, kind, 1)
    g = Q.group_rows(ids.to(dtype).cuda(), adapters)
    w = g.words.cpu().numpy()
    of = np.where((ids.numpy() >= 0) & (ids.numpy() < adapters), ids.numpy(), adapters)
    assert g.rows == rows and g.adapters == adapters
    assert np.array_equal(w[:rows], np.argsort(of, kind="stable"))
    counts = np.bincount(of, minlength=adapters + 1)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    assert np.array_equal(w[rows:rows + adapters + 2], offsets)
    first = w[rows + adapters + 2:rows + 2 * adapters + 3]
    slots = w[(rows + 2 * adapters + 6) // 4 * 4:].reshape(-1, 4)
    assert len(slots) == rows // 64 + min(rows, adapters + 1)
    want = {}
    for a in np.nonzero(counts)[0]:
        for j in range(-(-counts[a] // 64)):
            want[int(first[a]) + j] = (int(a), int(offsets[a]) + 64 * j, int(min(64, counts[a] - 64 * j)), j)
    assert {i: tuple(map(int, s)) for i, s in enumerate(slots) if s[0] >= 0} == want


SIZES = [(1, 1, 1, 1, 1), (1, 4, 8, 64, 40), (3, 2, 16, 8, 300), (16, 5, 16, 500, 256), (17, 1, 4, 64, 65), (64, 48, 16, 1024, 1024), (65, 3, 33, 1000, 777), (200, 4, 64, 2048, 512),
         (130, 2, 128, 264, 1030), (1000, 6, 12, 333, 515), (700, 3, 100, 96, 2000), (2500, 2, 16, 256, 256), (90, 90, 32, 4100, 130)]


@pytest.mark.parametrize("rows,adapters,rank,k,n", SIZES)
@pytest.mark.parametrize("dtype,y_dtype,kind", [(BF16, BF16, "mixed"), (F16, F16, "runs"), (BF16, F32, "one"), (F16, F32, "mixed"), (BF16, F16, "runs")])
def test_forward(rows, adapters, rank, k, n, dtype, y_dtype, kind):
    say("add_adapters", rows, adapters, rank, k, n, dtype, y_dtype, kind)
    y, x, A, B, s = operands(rows, adapters, rank, k, n, dtype, y_dtype, rows + rank)
    check(y, x, A, B, ids_of(rows, adapters, kind, rows), s)


@pytest.mark.parametrize("rows,adapters,rank,k,n", SIZES)
@pytest.mark.parametrize("dtype,dx_dtype,grad,kind", [(BF16, BF16, F32, "mixed"), (F16, F16, F32, "runs"), (BF16, F32, BF16, "one"), (F16, None, F16, "mixed"), (BF16, None, F32, "none")])
def test_backward(rows, adapters, rank, k, n, dtype, dx_dtype, grad, kind):
    say("add_adapters_backward", rows, adapters, rank, k, n, dtype, dx_dtype, grad, kind)
    y, x, A, B, s = operands(rows, adapters, rank, k, n, dtype, dtype, rows + rank)
    ids = ids_of(rows, adapters, kind, rows)
    u = Q.add_adapters(y, x, A, B, Q.group_rows(ids.cuda(), adapters), s, keep=True)[1]
    dy = values((rows, n), dtype, 77, n ** -0.5)
    check_backward(dy, x, u, A, B, ids, s, None if dx_dtype is None else values((rows, k), dx_dtype, 78, n ** -0.5), grad)


def test_gradients_of_many_rows():
    """Groups whose sums are shared out between workgroups, beside groups of few rows and of none."""
    say("add_adapters_backward many rows")
    rows, adapters, rank, k, n = 9000, 9, 16, 256, 384
    ids = torch.cat([torch.full((5000,), 2), torch.full((300,), 7), torch.full((3600,), 4), torch.full((100,), 0)])[torch.randperm(rows, generator=torch.Generator().manual_seed(2))]
    y, x, A, B, s = operands(rows, adapters, rank, k, n, BF16, BF16, 5)
    u = Q.add_adapters(y, x, A, B, Q.group_rows(ids.cuda(), adapters), s, keep=True)[1]
    _, dA, dB = check_backward(values((rows, n), BF16, 6, n ** -0.5), x, u, A, B, ids, s, None)
    for i in (1, 3, 5, 6, 8):
        assert (dA[i] == 0).all() and (dB[i] == 0).all()


@pytest.mark.parametrize("rows", [17000, 40000])
def test_many_rows(rows):
    """More rows than a group's registers hold ids of, forward against 64 bits, and gradients of sums in many parts."""
    say("add_adapters many rows", rows)
    adapters, rank, k, n = 5, 8, 64, 72
    y, x, A, B, s = operands(rows, adapters, rank, k, n, BF16, BF16, 50)
    ids = ids_of(rows, adapters, "mixed", 51)
    _, u, _ = check(y, x, A, B, ids, s)
    check_backward(values((rows, n), BF16, 52, n ** -0.5), x, u, A, B, ids, s, None)


def test_small_gradients_of_fp16():
    """Gradients far below what fp16 resolves beside ordinary ones: u and v keep their exponents."""
    say("add_adapters_backward small gradients")
    y, x, A, B, s = operands(100, 2, 16, 128, 192, F16, F16, 9)
    ids = ids_of(100, 2, "mixed", 9)
    u = values((100, 16), F32, 10, 3e-7)
    check_backward(values((100, 192), F16, 11, 1e-3), x, u, A, (B * 1e-3).contiguous(), ids, s, None)
    u = values((100, 16), F32, 12, 1e9)
    check_backward(values((100, 192), F16, 11, 1e-3), x, u, A, B, ids, s, None)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_strides_addresses_dimensions_and_in_place(dtype):
    say("add_adapters strides", dtype)
    rows, adapters, rank, k, n = 60, 4, 16, 300, 203
    A, B = values((adapters, rank, k), dtype, 13, k ** -0.5), values((adapters, rank, n), dtype, 14)
    ids = ids_of(rows, adapters, "mixed", 15)
    x, y = values((3, 20, k), dtype, 16, gap=5, offset=1), values((3, 20, n), dtype, 17, gap=3, offset=3)
    want, u, groups = check(y, x, A, B, ids, None)
    room = torch.full((rows, n + 9), 7.0, dtype=dtype, device="cuda")
    out = room[:, 2:2 + n].view(3, 20, n) if room[:, 2:2 + n].is_contiguous() else room[:, 2:2 + n].unflatten(0, (3, 20))
    assert Q.add_adapters(y, x, A, B, groups, out=out) is out
    assert torch.equal(out, want) and (room[:, :2] == 7).all() and (room[:, 2 + n:] == 7).all()
    gaps = y.new_empty(0).set_(y.untyped_storage(), 0, (y.untyped_storage().size() // 2,)).clone()
    assert Q.add_adapters(y, x, A, B, groups, out=y) is y
    assert torch.equal(y, want)
    after = y.new_empty(0).set_(y.untyped_storage(), 0, (y.untyped_storage().size() // 2,))
    assert torch.equal(torch.isnan(after), torch.isnan(gaps))       # (what lies between the rows is left as it was)
    dy = values((3, 20, n), dtype, 18, gap=1, offset=5)
    check_backward(dy, x, u, A, B, ids, None, values((3, 20, k), F32, 19, gap=4, offset=1))


def test_rows_of_no_adapter_keep_their_bits():
    say("add_adapters none")
    y, x, A, B, s = operands(150, 3, 8, 64, 100, BF16, BF16, 20)
    x[:, 3] = float("nan")
    y[0, 0], y[1, 1] = float("inf"), float("nan")
    ids = ids_of(150, 3, "none", 21)
    out, u = Q.add_adapters(y, x, A, B, Q.group_rows(ids.cuda(), 3), s, keep=True)
    assert torch.equal(out.view(torch.int16), y.view(torch.int16)) and (u == 0).all()
    ids[7] = 1
    out = Q.add_adapters(y, x, A, B, Q.group_rows(ids.cuda(), 3), s)
    assert torch.isnan(out[7]).all()
    out[7] = y[7]
    assert torch.equal(out.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("rank", [8, 40])
def test_padding_of_a_rank_and_of_rows_adds_nothing(rank):
    """What lies behind a factor's last row, column and adapter is nobody's: NaN there changes nothing."""
    say("add_adapters padding", rank)
    y, x, A, B, s = operands(37, 3, rank, 100, 131, BF16, BF16, 22)
    ids = ids_of(37, 3, "mixed", 23)
    want = Q.add_adapters(y, x, A, B, Q.group_rows(ids.cuda(), 3), s)
    wide_A, wide_B = torch.full((4, rank, 100), float("nan"), dtype=BF16, device="cuda"), torch.full((4, rank, 131), float("nan"), dtype=BF16, device="cuda")
    wide_A[:3], wide_B[:3] = A, B
    assert torch.equal(Q.add_adapters(y, x, wide_A[:3], wide_B[:3], Q.group_rows(ids.cuda(), 3), s), want)


def test_backward_against_differences():
    say("add_adapters differences")
    y, x, A, B, s = operands(12, 3, 4, 24, 30, BF16, F32, 24)
    ids = ids_of(12, 3, "mixed", 25)
    groups = Q.group_rows(ids.cuda(), 3)
    _, u = Q.add_adapters(y, x, A, B, groups, s, keep=True)
    dy = values((12, 30), BF16, 26)
    dx, dA, dB = (R.f64(t) for t in Q.add_adapters_backward(dy, x, u, A, B, groups, s, dx=torch.zeros(12, 24, device="cuda")))
    X, AA, BB, D, S = (R.f64(t) for t in (x, A, B, dy, s))

    def value(X, AA, BB):
        return (L.adapters(np.zeros((12, 30)), X, AA, BB, ids.numpy(), S, 3)[0][0] * D).sum()

    rng = np.random.default_rng(3)
    for _ in range(8):
        a, b, c, step = rng.standard_normal(X.shape), rng.standard_normal(AA.shape), rng.standard_normal(BB.shape), 1e-5
        got = (dx * a).sum() + (dA * b).sum() + (dB * c).sum()
        want = (value(X + step * a, AA + step * b, BB + step * c) - value(X - step * a, AA - step * b, BB - step * c)) / (2 * step)
        assert abs(got - want) <= 1e-5 * np.sqrt((dx ** 2).sum() + (dA ** 2).sum() + (dB ** 2).sum())


def everything(y, x, A, B, ids, s, dy):
    groups = Q.group_rows(ids, len(A))
    out, u = Q.add_adapters(y, x, A, B, groups, s, keep=True)
    return (out, u, *Q.add_adapters_backward(dy, x, u, A, B, groups, s, dx=x))


@pytest.mark.parametrize("rows,adapters", [(40, 30), (5000, 3)])
def test_the_same_bits_again_and_on_another_stream(rows, adapters):
    say("add_adapters again", rows, adapters)
    y, x, A, B, s = operands(rows, adapters, 16, 512, 320, BF16, BF16, 27)
    ids, dy = ids_of(rows, adapters, "mixed", 28).cuda(), values((rows, 320), BF16, 29)
    first = everything(y, x, A, B, ids, s, dy)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = everything(y, x, A, B, ids, s, dy)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_a_captured_pass():
    """A graph takes the ids that lie there when it is replayed."""
    say("add_adapters captured")
    y, x, A, B, s = operands(600, 5, 16, 512, 320, BF16, BF16, 30)
    ids, dy = ids_of(600, 5, "mixed", 31).cuda(), values((600, 320), BF16, 32)
    everything(y, x, A, B, ids, s, dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = everything(y, x, A, B, ids, s, dy)
    for seed, kind in ((33, "mixed"), (34, "runs"), (35, "one"), (36, "none")):
        x.copy_(values((600, 512), BF16, seed))
        ids.copy_(ids_of(600, 5, kind, seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, everything(y, x, A, B, ids, s, dy)))


def test_through_ctypes(monkeypatch):
    say("add_adapters ctypes")
    y, x, A, B, s = operands(70, 4, 24, 130, 90, F16, F32, 37)
    ids, dy = ids_of(70, 4, "mixed", 38).cuda(), values((70, 90), F16, 39)
    want = everything(y, x, A, B, ids, s, dy)
    monkeypatch.setattr(Q.ops, "_native_module", False)
    assert all(torch.equal(a, b) for a, b in zip(want, everything(y, x, A, B, ids, s, dy)))


def test_no_rows():
    say("add_adapters no rows")
    A, B = values((3, 8, 64), BF16, 40), values((3, 8, 32), BF16, 41)
    x, y = torch.empty(0, 64, dtype=BF16, device="cuda"), torch.empty(0, 32, dtype=BF16, device="cuda")
    groups = Q.group_rows(torch.empty(0, dtype=torch.int32, device="cuda"), 3)
    out, u = Q.add_adapters(y, x, A, B, groups, keep=True)
    assert out.shape == (0, 32) and u.shape == (0, 8)
    dx, dA, dB = Q.add_adapters_backward(y, x, u, A, B, groups)
    assert dx.shape == (0, 64) and (dA == 0).all() and (dB == 0).all()


def test_offsets_beyond_32_bits():
    """Rows of x and y, and factors, whose offsets pass 2^32 bytes and elements."""
    say("add_adapters offsets")
    rows, k = (1 << 20) + 70, 4128
    x = torch.zeros(rows, k, dtype=BF16, device="cuda")
    x[-70:] = values((70, k), BF16, 42)
    A, B = values((2, 4, k), BF16, 43, k ** -0.5), values((2, 4, k), BF16, 44)
    ids = torch.full((rows,), -1, dtype=torch.int32)
    ids[-70:] = ids_of(70, 2, "mixed", 45)
    out = Q.add_adapters(x, x, A, B, Q.group_rows(ids.cuda(), 2))
    want = Q.add_adapters(x[-70:], x[-70:], A, B, Q.group_rows(ids[-70:].cuda(), 2))
    # (the columns are split between workgroups for few rows and not for many: another order of the same fp32 sums)
    assert torch.allclose(out[-70:].float(), want.float(), rtol=2 ** -7, atol=1e-4) and (out[:-70] == 0).all()
    del out
    many = torch.zeros(40000, 16, 4096, dtype=BF16, device="cuda")
    many[-1] = values((16, 4096), BF16, 46, 1 / 64)
    xs, ys = values((5, 4096), BF16, 47), values((5, 4096), BF16, 48)
    got = Q.add_adapters(ys, xs, many, many, Q.group_rows(torch.full((5,), 39999, dtype=torch.int64, device="cuda"), 40000))
    one = Q.add_adapters(ys, xs, many[-1:], many[-1:], Q.group_rows(torch.zeros(5, dtype=torch.int64, device="cuda"), 1))
    assert torch.equal(got, one)
