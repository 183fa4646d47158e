"""What the training entries refuse, before anything is launched: no device is needed."""
import pytest
import torch

import qgemm_amd as Q
from qgemm_amd.lib import load_library

F32, BF16, F16, I8, F8, I32 = Q.DT_F32, Q.DT_BF16, Q.DT_F16, Q.DT_I8, Q.DT_F8E4M3, Q.DT_I32
P = 1 << 32
INVALID, UNSUPPORTED, TOO_LARGE = 1, 2, 9


def norm(x_dt=BF16, y_dt=BF16, p_dt=F32, q_dt=I8, x=P, ldx=64, w=P, b=P, eps=1e-5, y=P, ldy=64, q=P, ldq=64, s=P, rows=4, cols=64):
    return load_library().qgemm_layer_norm(x_dt, y_dt, p_dt, q_dt, x, ldx, w, b, eps, y, ldy, P, P, q, ldq, s, rows, cols, None)


def backward(dy_dt=BF16, x_dt=BF16, dx_dt=BF16, p_dt=F32, dy=P, lddy=64, x=P, ldx=64, s=None, mean=P, rstd=P, w=P, dx=P, lddx=64, dw=P, db=P, rows=4, cols=64):
    return load_library().qgemm_layer_norm_backward(dy_dt, x_dt, dx_dt, p_dt, dy, lddy, x, ldx, s, mean, rstd, w, dx, lddx, dw, db, rows, cols, None)


def gradient(dy_dt=BF16, q_dt=I8, dw_dt=F32, p_dt=F32, dy=P, lddy=32, q=P, ldq=64, s=P, w=P, b=P, dw=P, lddw=64, rows=4, n=32, cols=64):
    return load_library().qgemm_weight_gradient(dy_dt, q_dt, dw_dt, p_dt, dy, lddy, q, ldq, s, w, b, dw, lddw, P, rows, n, cols, None)


def checkpoint(x_dt=BF16, q_dt=I8, x=P, ldx=64, rows=4, cols=64, q=P, ldq=64, s=P):
    return load_library().qgemm_checkpoint(x_dt, q_dt, x, ldx, rows, cols, q, ldq, s, None)


def restore(q_dt=I8, x_dt=BF16, q=P, ldq=64, s=P, rows=4, cols=64, x=P, ldx=64):
    return load_library().qgemm_restore(q_dt, x_dt, q, ldq, s, rows, cols, x, ldx, None)


@pytest.mark.parametrize("entry,status,arguments", [
    (norm, UNSUPPORTED, [dict(x_dt=I8), dict(y_dt=I32), dict(p_dt=F8), dict(q_dt=BF16), dict(x_dt=17)]),
    (norm, INVALID, [dict(x=None), dict(y=None), dict(cols=0), dict(ldx=63), dict(ldy=63), dict(ldq=63), dict(w=None), dict(eps=-1.0),
                     dict(eps=float("nan")), dict(s=None), dict(q=None)]),
    (norm, TOO_LARGE, [dict(rows=1 << 31), dict(cols=1 << 31)]),
    (backward, UNSUPPORTED, [dict(dy_dt=I8), dict(x_dt=I32), dict(dx_dt=F8), dict(p_dt=I8)]),
    (backward, INVALID, [dict(dy=None), dict(x=None), dict(dx=None), dict(rstd=None), dict(mean=None), dict(x_dt=I8), dict(cols=0), dict(lddy=63), dict(ldx=63),
                         dict(lddx=63)]),
    (backward, TOO_LARGE, [dict(rows=1 << 31), dict(cols=1 << 31)]),
    (gradient, UNSUPPORTED, [dict(dy_dt=F32), dict(dy_dt=I8), dict(q_dt=BF16), dict(dw_dt=I32), dict(p_dt=I8)]),
    (gradient, INVALID, [dict(dy=None), dict(q=None), dict(s=None), dict(dw=None), dict(cols=0), dict(lddy=31), dict(ldq=63), dict(lddw=63), dict(w=None)]),
    (gradient, TOO_LARGE, [dict(rows=1 << 31), dict(cols=1 << 31), dict(n=1 << 31)]),
    (checkpoint, UNSUPPORTED, [dict(x_dt=I8), dict(q_dt=F16)]),
    (checkpoint, INVALID, [dict(x=None), dict(q=None), dict(s=None), dict(ldx=63), dict(ldq=63)]),
    (checkpoint, TOO_LARGE, [dict(rows=1 << 31), dict(cols=1 << 31)]),
    (restore, UNSUPPORTED, [dict(q_dt=BF16), dict(x_dt=I8)]),
    (restore, INVALID, [dict(x=None), dict(q=None), dict(s=None), dict(ldx=63), dict(ldq=63)]),
    (restore, TOO_LARGE, [dict(rows=1 << 31), dict(cols=1 << 31)]),
])
def test_statuses(entry, status, arguments):
    for a in arguments:
        assert entry(**a) == status, a


def test_nothing_to_do_needs_nothing():
    assert norm(rows=0, x=None, y=None) == 0
    assert backward(rows=0, dy=None, x=None, dx=None, rstd=None, mean=None, dw=None, db=None) == 0
    assert gradient(n=0, dw=None) == 0
    assert checkpoint(rows=0, x=None) == 0 and restore(cols=0, q=None) == 0


def test_host_tensors_are_refused():
    x, q, s, v = torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 1), torch.zeros(4)
    for call in (lambda: Q.layer_norm(x), lambda: Q.layer_norm_backward(x, x, v, v), lambda: Q.checkpoint(x), lambda: Q.restore(q, s),
                 lambda: Q.weight_gradient(x.bfloat16(), q, s)):
        with pytest.raises(ValueError, match="device tensors"):
            call()


@pytest.mark.gpu
def test_tensors_that_do_not_fit():
    f = lambda *shape, dtype=torch.float32: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    x, q, s, v, w = f(4, 64, dtype=torch.bfloat16), f(4, 64, dtype=torch.int8), f(4, 1), f(4), f(64)
    bad_type = [lambda: Q.layer_norm(f(4, 64, dtype=torch.int8)), lambda: Q.layer_norm(x, w.double()), lambda: Q.layer_norm(x, keep=torch.bfloat16),
                lambda: Q.layer_norm(x, out_dtype=torch.int8), lambda: Q.checkpoint(x, torch.uint8), lambda: Q.checkpoint(q), lambda: Q.restore(x, s),
                lambda: Q.restore(q, s, torch.int8), lambda: Q.restore(q, s.bfloat16()), lambda: Q.weight_gradient(f(4, 8), q, s),
                lambda: Q.weight_gradient(x, x, s), lambda: Q.layer_norm_backward(x, x.double(), v, v),
                lambda: Q.weight_gradient(x, q.view(torch.uint8).view(torch.float8_e4m3fnuz), s)]
    bad_value = [lambda: Q.layer_norm(x.t()), lambda: Q.layer_norm(x[0, 0]), lambda: Q.layer_norm(x, w[:63]), lambda: Q.layer_norm(x, None, w),
                 lambda: Q.layer_norm(x, w, w.bfloat16()), lambda: Q.layer_norm(x[:1].expand(4, 64)), lambda: Q.layer_norm(x, w.cpu()),
                 lambda: Q.layer_norm(f(3, 4, 8).transpose(0, 1)), lambda: Q.layer_norm_backward(x, x, None, v), lambda: Q.layer_norm_backward(x, x[:3], v, v),
                 lambda: Q.layer_norm_backward(x, q, None, v), lambda: Q.layer_norm_backward(x, x, v, v, None, s), lambda: Q.layer_norm_backward(x, x, v, v[:3]),
                 lambda: Q.restore(q, s[:3]), lambda: Q.weight_gradient(x[:3], q, s), lambda: Q.weight_gradient(x, q, s, None, w),
                 lambda: Q.weight_gradient(x, q, f(4, 2)), lambda: Q.checkpoint(f(4, 0))]
    for call in bad_type:
        with pytest.raises(TypeError):
            call()
    for call in bad_value:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(Q.QgemmError, match="INVALID_ARG"):
        Q.layer_norm(x, eps=-1.0)
