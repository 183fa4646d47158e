"""What the entries beside the products refuse, before anything is launched, and the launches that they make: no device is needed but for the last test."""
import ctypes as C

import pytest
import torch

import qgemm_amd as Q
from qgemm_amd.lib import load_library
from tests import host_runtime

F32, BF16, F16, I8, F8, I32 = Q.DT_F32, Q.DT_BF16, Q.DT_F16, Q.DT_I8, Q.DT_F8E4M3, Q.DT_I32
P = 1 << 32
INVALID, UNSUPPORTED, TOO_LARGE = 1, 2, 9


def norm(x_dt=BF16, r_dt=BF16, y_dt=BF16, p_dt=F32, q_dt=I8, x=P, ldx=64, r=P, ldr=64, w=P, eps=1e-6, h=P, ldh=64, y=P, ldy=64, q=P, ldq=64, s=P, rows=4, cols=64):
    return load_library().qgemm_rms_norm(x_dt, r_dt, y_dt, p_dt, q_dt, x, ldx, r, ldr, w, eps, h, ldh, y, ldy, P, q, ldq, s, rows, cols, None)


def norm_backward(dy_dt=BF16, h_dt=BF16, dh_dt=F32, dx_dt=BF16, p_dt=F32, dy=P, lddy=64, h=P, ldh=64, rstd=P, w=P, dh=P, lddh=64, dx=P, lddx=64, dw=P, rows=4, cols=64):
    return load_library().qgemm_rms_norm_backward(dy_dt, h_dt, dh_dt, dx_dt, p_dt, dy, lddy, h, ldh, rstd, w, dh, lddh, dx, lddx, dw, rows, cols, None)


def group(bytes=4, ids=P, rows=4, adapters=2, groups=P):
    return load_library().qgemm_group_rows(bytes, ids, rows, adapters, groups, None)


def add(dt=BF16, y_dt=BF16, y=P, ldy=32, x=P, ldx=64, A=P, B=P, groups=P, out=P, ldo=32, rows=4, adapters=2, rank=8, k=64, n=32):
    return load_library().qgemm_add_adapters(dt, y_dt, y, ldy, x, ldx, A, B, P, groups, out, ldo, P, rows, adapters, rank, k, n, None)


def add_backward(dt=BF16, dx_dt=BF16, g_dt=F32, dy=P, lddy=32, x=P, ldx=64, u=P, A=P, B=P, groups=P, dx0=P, lddx0=64, dx=2 * P, lddx=64, dA=P, dB=P, rows=4, adapters=2, rank=8,
                 k=64, n=32):
    return load_library().qgemm_add_adapters_backward(dt, dx_dt, g_dt, dy, lddy, x, ldx, u, A, B, P, groups, dx0, lddx0, dx, lddx, dA, dB, rows, adapters, rank, k, n, None)


def log_prob(dt=BF16, bytes=8, x=P, ld=64, t=P, top=4, logp=P, entropy=P, lse=P, values=P, indices=P, rows=4, cols=64):
    return load_library().qgemm_log_probabilities(dt, bytes, x, ld, t, top, logp, entropy, lse, values, indices, rows, cols, None)


def log_prob_backward(dt=BF16, out=BF16, bytes=8, x=P, ld=64, t=P, lse=P, entropy=P, a=P, b=P, dx=P, ldd=64, rows=4, cols=64):
    return load_library().qgemm_log_probabilities_backward(dt, out, bytes, x, ld, t, lse, entropy, a, b, dx, ldd, rows, cols, None)


@pytest.mark.parametrize("entry,status,arguments", [
    (norm, UNSUPPORTED, [dict(x_dt=I8), dict(r_dt=I32), dict(y_dt=F8), dict(p_dt=F8), dict(q_dt=BF16), dict(x_dt=17)]),
    (norm, INVALID, [dict(x=None), dict(y=None, q=None, s=None), dict(cols=0), dict(ldx=63), dict(ldr=63), dict(ldh=63), dict(ldy=63), dict(ldq=63), dict(eps=-1.0),
                     dict(eps=float("nan")), dict(s=None), dict(q=None), dict(h=None), dict(r=None)]),
    (norm, TOO_LARGE, [dict(rows=1 << 31), dict(cols=1 << 31)]),
    (norm_backward, UNSUPPORTED, [dict(dy_dt=I8), dict(h_dt=I8), dict(dh_dt=I32), dict(dx_dt=F8), dict(p_dt=I8)]),
    (norm_backward, INVALID, [dict(dy=None), dict(h=None), dict(dx=None), dict(rstd=None), dict(cols=0), dict(lddy=63), dict(ldh=63), dict(lddh=63), dict(lddx=63)]),
    (norm_backward, TOO_LARGE, [dict(rows=1 << 31), dict(cols=1 << 31), dict(cols=(1 << 31) - 1, lddy=1 << 31, ldh=1 << 31, lddh=1 << 31, lddx=1 << 31)]),
    (group, UNSUPPORTED, [dict(bytes=2)]),
    (group, INVALID, [dict(ids=None), dict(adapters=0), dict(groups=None), dict(groups=P + 8)]),
    (group, TOO_LARGE, [dict(rows=1 << 28), dict(adapters=65536)]),
    (add, UNSUPPORTED, [dict(dt=F32), dict(dt=F8), dict(y_dt=I32)]),
    (add, INVALID, [dict(y=None), dict(x=None), dict(A=None), dict(B=None), dict(groups=None), dict(groups=P + 8), dict(out=None), dict(ldy=31), dict(ldx=63), dict(ldo=31),
                    dict(ldo=33), dict(adapters=0), dict(rank=0), dict(k=0), dict(n=0)]),
    (add, TOO_LARGE, [dict(rows=1 << 28), dict(adapters=65536), dict(rank=129), dict(k=1 << 23), dict(n=1 << 23)]),
    (add_backward, UNSUPPORTED, [dict(dt=F32), dict(dx_dt=I8), dict(g_dt=I32)]),
    (add_backward, INVALID, [dict(dy=None), dict(x=None), dict(u=None), dict(A=None), dict(B=None), dict(groups=None), dict(groups=P + 8), dict(dx=None), dict(lddy=31), dict(ldx=63),
                             dict(lddx=63), dict(lddx0=63), dict(dx=P, lddx=65), dict(adapters=0), dict(rank=0), dict(k=0), dict(n=0)]),
    (add_backward, TOO_LARGE, [dict(rows=1 << 28), dict(adapters=65536), dict(rank=129), dict(k=1 << 23), dict(n=1 << 23)]),
    (log_prob, UNSUPPORTED, [dict(dt=I8), dict(bytes=1)]),
    (log_prob, INVALID, [dict(x=None), dict(t=None), dict(logp=None), dict(entropy=None), dict(lse=None), dict(values=None), dict(indices=None), dict(ld=63), dict(cols=0), dict(top=-1),
                         dict(top=5, cols=4)]),
    (log_prob, TOO_LARGE, [dict(rows=1 << 31), dict(cols=1 << 31), dict(top=33)]),
    (log_prob_backward, UNSUPPORTED, [dict(dt=I8), dict(out=I32), dict(bytes=1)]),
    (log_prob_backward, INVALID, [dict(x=None), dict(t=None), dict(lse=None), dict(entropy=None), dict(a=None), dict(dx=None), dict(ld=63), dict(ldd=63), dict(cols=0)]),
    (log_prob_backward, TOO_LARGE, [dict(rows=1 << 31), dict(cols=1 << 31)]),
])
def test_statuses(entry, status, arguments):
    for a in arguments:
        assert entry(**a) == status, a


def test_nothing_to_do_needs_nothing():
    assert norm(rows=0, x=None, y=None, q=None, s=None) == 0
    assert norm_backward(rows=0, dy=None, h=None, dx=None, rstd=None, dw=None) == 0
    assert add(rows=0, y=None, x=None, out=None) == 0 and add_backward(rows=0, dA=None, dB=None, groups=None) == 0
    assert log_prob(rows=0, x=None) == 0 and log_prob_backward(rows=0, x=None) == 0


def test_words_of_groups():
    words = C.c_size_t()
    f = load_library().qgemm_group_rows_words
    assert f(0, 1, C.byref(words)) == 0 and words.value == 8
    assert f(1000, 7, C.byref(words)) == 0 and words.value == 1020 + 4 * (15 + 8)
    assert f(4, 0, C.byref(words)) == INVALID and f(4, 1, None) == INVALID and f(4, 65536, C.byref(words)) == TOO_LARGE and f(1 << 28, 1, C.byref(words)) == TOO_LARGE


def test_host_tensors_are_refused():
    x, v, t = torch.zeros(4, 64).bfloat16(), torch.zeros(4), torch.zeros(4, dtype=torch.int64)
    groups = Q.RowGroups(4, 2, torch.zeros(40, dtype=torch.int32))
    A = torch.zeros(2, 8, 64).bfloat16()
    for call in (lambda: Q.rms_norm(x), lambda: Q.rms_norm_backward(x, x, v), lambda: Q.group_rows(t, 2), lambda: Q.add_adapters(x, x, A, A, groups),
                 lambda: Q.add_adapters_backward(x, x, torch.zeros(4, 8), A, A, groups), lambda: Q.log_probabilities(x, t),
                 lambda: Q.log_probabilities_backward(x, t, v, v, v)):
        with pytest.raises(ValueError, match="device tensors"):
            call()


def test_no_launch_is_larger_than_the_runtime_takes(tmp_path_factory):
    """Fewer than 2^32 threads across and 2^16 workgroups down, and no more workspace than a stream's own block has, whatever size is not refused."""
    host_runtime.run(tmp_path_factory, """
import random
P, OK, TOO_LARGE = 1 << 40, 0, 9
rng = random.Random(3)
runtime.host_budget(1 << 62)
def check(what, status, most=128 << 20):
    made, took = [], 0
    for e in events():
        m = re.match(r"launch _ZN5qgemm[0-9]+([a-z0-9_]+?_kernel).* grid ([0-9]+) ([0-9]+) block ([0-9]+)", e)
        if m:
            made.append((m[1], *map(int, m.groups()[1:])))
        if e.startswith("malloc"):
            took = max(took, int(e.split()[1]))
    assert status in (OK, TOO_LARGE) and bool(made) == (status == OK), (what, status, made)
    for name, x, y, block in made:
        assert 0 < x * block < 1 << 32 and 0 < y < 1 << 16, (what, name, x, y, block)
    return took
edges = [1, 7, 8, 64, 65, 16384, 16385, 1 << 18, 1 << 24, (1 << 23) - 256, 1 << 27, (1 << 28) - 1, 1 << 28, 1 << 30, (1 << 31) - 129, (1 << 31) - 128, (1 << 31) - 127, (1 << 31) - 1, 1 << 31]
size = lambda most=31: rng.choice(edges) if rng.random() < 0.3 else int(2 ** rng.uniform(0, most))
for _ in range(2000):
    rows, cols = size(), size()
    check(("norm", rows, cols), lib.qgemm_rms_norm(BF16, BF16, BF16, F32, I8, P, cols, P, cols, P, 1e-6, P, cols, P, cols, P, P, cols, P, rows, cols, 0))
    check(("norm backward", rows, cols), lib.qgemm_rms_norm_backward(BF16, BF16, F32, BF16, F32, P, cols, P, cols, P, P, P, cols, P, cols, P, rows, cols, 0))
    top = rng.choice([0, 1, 20, 32])
    check(("log", rows, cols, top), lib.qgemm_log_probabilities(BF16, 8, P, cols, P, min(top, cols), P, P, P, P, P, rows, cols, 0))
    check(("log backward", rows, cols), lib.qgemm_log_probabilities_backward(BF16, BF16, 8, P, cols, P, P, P, P, P, P, cols, rows, cols, 0))
    adapters, rank, k, n = int(2 ** rng.uniform(0, 16)), rng.randint(1, 128), size(24), size(24)
    check(("group", rows, adapters), lib.qgemm_group_rows(4, P, rows, adapters, P, 0))
    check(("add", rows, adapters, rank, k, n), lib.qgemm_add_adapters(BF16, BF16, P, n, P, k, P, P, P, P, 2 * P, n, P, rows, adapters, rank, k, n, 0))
    check(("add backward", rows, adapters, rank, k, n),
          lib.qgemm_add_adapters_backward(BF16, BF16, F32, P, n, P, k, P, P, P, P, P, P, k, 2 * P, k, P, P, rows, adapters, rank, k, n, 0))
for _ in range(300):
    rows, cols, adapters, rank = int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 10)), rng.randint(1, 128)
    lib.qgemm_shutdown()
    events()
    for call in (lambda: lib.qgemm_rms_norm_backward(BF16, BF16, F32, BF16, F32, P, cols, P, cols, P, P, P, cols, P, cols, P, rows, cols, 0),
                 lambda: lib.qgemm_log_probabilities(BF16, 8, P, cols, P, min(20, cols), P, P, P, P, P, rows, cols, 0)):
        assert check((rows, cols), call()) <= 128 << 20, (rows, cols)
""")


@pytest.mark.gpu
def test_tensors_that_do_not_fit():
    f = lambda *shape, dtype=torch.bfloat16: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    x, v, w, t = f(4, 64), f(4, dtype=torch.float32), f(64, dtype=torch.float32), f(4, dtype=torch.int64)
    y, A, B, u = f(4, 32), f(2, 8, 64), f(2, 8, 32), f(4, 8, dtype=torch.float32)
    g, other = Q.group_rows(t, 2), Q.group_rows(t, 3)
    add, back = Q.add_adapters, Q.add_adapters_backward
    bad_type = [lambda: Q.rms_norm(f(4, 64, dtype=torch.int8)), lambda: Q.rms_norm(x, w.double()), lambda: Q.rms_norm(x, residual=x.double()), lambda: Q.rms_norm(x, codes=torch.bfloat16),
                lambda: Q.rms_norm(x, out_dtype=torch.int8), lambda: Q.rms_norm_backward(x, x.double(), v), lambda: Q.rms_norm_backward(x, x, v.double()),
                lambda: Q.rms_norm_backward(x, x, v, dh=x.double()), lambda: Q.group_rows(t.float(), 2), lambda: add(y, x.float(), A, B, g), lambda: add(y, x, A.half(), B, g),
                lambda: add(y, x, A, B.float(), g), lambda: add(y.double(), x, A, B, g), lambda: add(y, x, A, B, t), lambda: add(y, x, A, B, g, f(2)), lambda: add(y, x, A, B, g, out=y.float()),
                lambda: back(y.half(), x, u, A, B, g), lambda: back(y, x, u.half(), A, B, g), lambda: back(y, x, u, A, B, g, grad_dtype=torch.int8), lambda: back(y, x, u, A, B, g, dx=x.double()),
                lambda: Q.log_probabilities(x.double(), t), lambda: Q.log_probabilities(x, t.float()), lambda: Q.log_probabilities_backward(x, t, v.half(), v, v),
                lambda: Q.log_probabilities_backward(x, t, v, v, v, out_dtype=torch.int8)]
    bad_value = [lambda: Q.rms_norm(x.t()), lambda: Q.rms_norm(x, w[:63]), lambda: Q.rms_norm(x, residual=x[:3]), lambda: Q.rms_norm(x, residual=f(4, 65)), lambda: Q.rms_norm(x, store_y=False),
                 lambda: Q.rms_norm(x, w.cpu()), lambda: Q.rms_norm(x[:1].expand(4, 64)), lambda: Q.rms_norm_backward(x, x[:3], v), lambda: Q.rms_norm_backward(x, x, v[:3]),
                 lambda: Q.rms_norm_backward(x, x, v, dh=f(4, 63)), lambda: Q.group_rows(t[::2], 2), lambda: Q.group_rows(t, -1), lambda: Q.group_rows(t.cpu(), 2),
                 lambda: add(y, x, A, B, other), lambda: add(y, x[:3], A, B, g), lambda: add(y[:3], x, A, B, g), lambda: add(y, x, A[:1], B, g), lambda: add(y, x, A, B[:, :4], g),
                 lambda: add(y, x, A.transpose(0, 1), B, g), lambda: add(y, x, A, B.flatten(1), g), lambda: add(y, x, A, B, g, v), lambda: add(y, x, A, B, g, out=f(4, 33)),
                 lambda: add(y, x, A, B, g, out=y.view(2, 2, 32)), lambda: add(y, f(4, 60), A, B, g), lambda: back(x, x, u, A, B, g), lambda: back(y, x, u[:3], A, B, g),
                 lambda: back(y, x, u, A, B, g, dx=y), lambda: Q.log_probabilities(x, t[:3]), lambda: Q.log_probabilities(x, t, -1), lambda: Q.log_probabilities(x, t.cpu()),
                 lambda: Q.log_probabilities_backward(x, t, v[:3], v, v), lambda: Q.log_probabilities_backward(x, t, v, v, v, v[:3])]
    for native in (Q.ops._native(), False):
        saved, Q.ops._native_module = Q.ops._native_module, native
        try:
            for call in bad_type:
                with pytest.raises(TypeError):
                    call()
            for call in bad_value:
                with pytest.raises(ValueError):
                    call()
            for call in (lambda: Q.rms_norm(x, eps=-1.0), lambda: Q.group_rows(t, 0), lambda: Q.log_probabilities(f(4, 8), t, 9),
                         lambda: Q.log_probabilities_backward(x, t, v, None, v, v)):
                with pytest.raises(Q.QgemmError, match="INVALID_ARG"):
                    call()
            for call in (lambda: Q.group_rows(t, 65536), lambda: Q.log_probabilities(x, t, 33), lambda: add(y, x, f(2, 129, 64), f(2, 129, 32), g)):
                with pytest.raises(Q.QgemmError, match="TOO_LARGE"):
                    call()
        finally:
            Q.ops._native_module = saved
