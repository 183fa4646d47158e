"""Layer norm, activations in 8 bits and their gradients in 64 bits, from the formulas, with the error that fp32 sums may leave.

u = 2^-24 is half a last place of fp32.  A row's sum passes through at most 32 roundings on its way (eight elements of a lane one after
the other or as a tree, up to eight octets of a lane, six or ten exchanges between lanes and waves), each of no more than u
times the row's largest |term| per element: 32 u max|term| on a mean."""
import numpy as np
import torch

U = 2.0 ** -24
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
LEAST = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in HALF_STEP}
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def f64(t):
    """Values on the host in 64 bits (codes as the numbers they are)."""
    return t.detach().cpu().float().double().numpy() if t.dtype != torch.float64 else t.detach().cpu().numpy()


def stored(bound, ref, dtype):
    """`bound` on a value before it is rounded to dtype."""
    return bound * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * np.abs(ref) + LEAST[dtype]


def check(got, ref, bound, what=""):
    got = f64(got).reshape(ref.shape)
    err = np.abs(got - ref)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(err / bound):.3g} of the bound, at {np.argwhere(bad)[0]}"


def norm(x, w, b, eps):
    """y, mean, rstd, xhat and the bounds of y (before rounding), mean, rstd, xhat."""
    n = x.shape[-1]
    mean = x.mean(-1, keepdims=True)
    away = x - mean
    rstd = 1 / np.sqrt((away * away).mean(-1, keepdims=True) + eps)
    xhat = away * rstd
    top = np.abs(x).max(-1, keepdims=True)
    e_mean = 32 * U * top
    # a sum of squares of positive terms: 32 roundings of it, and each centred value is off by the mean's error and one rounding
    off = e_mean + U * (np.abs(away) + top)
    e_var = (34 * U * away * away + 2 * np.abs(away) * off + off * off).mean(-1, keepdims=True)
    e_rstd = rstd * (0.5 * e_var * rstd * rstd * (1 + e_var * rstd * rstd) + 4 * U)
    e_xhat = off * rstd * 2 + np.abs(away) * e_rstd + 2 * U * np.abs(xhat)
    y, e_y = xhat, e_xhat
    if w is not None:
        y, e_y = y * w, e_y * np.abs(w) + 2 * U * np.abs(y * w)
    if b is not None:
        y, e_y = y + b, e_y + 2 * U * (np.abs(y) + np.abs(b))
    return (y, mean, rstd, xhat), (e_y, e_mean, e_rstd, e_xhat)


def norm_gradients(dy, xhat, e_xhat, rstd, w):
    """dx, dw, db and their bounds (before rounding); rstd as it was handed over."""
    rows, n = dy.shape
    g = dy if w is None else dy * w
    a, b = g.mean(-1, keepdims=True), (g * xhat).mean(-1, keepdims=True)
    dx = rstd * (g - a - xhat * b)
    e_g = U * np.abs(g)
    e_a = e_g.mean(-1, keepdims=True) + 32 * U * np.abs(g).max(-1, keepdims=True)
    e_b = (e_g * np.abs(xhat) + np.abs(g) * e_xhat).mean(-1, keepdims=True) + 34 * U * np.abs(g * xhat).max(-1, keepdims=True)
    e_dx = rstd * (e_g + e_a + np.abs(xhat) * e_b + e_xhat * np.abs(b) + 4 * U * (np.abs(g) + np.abs(a) + np.abs(xhat * b))) + U * np.abs(dx)
    # over rows: no more than one sixteenth of them one after the other, and 64 partial sums behind that
    adds = rows / 16 + 80
    dw, db = (dy * xhat).sum(0), dy.sum(0)
    e_dw = adds * U * np.abs(dy * xhat).sum(0) + (np.abs(dy) * e_xhat).sum(0)
    return (dx, dw, db), (e_dx, e_dw, adds * U * np.abs(dy).sum(0))


def blocks(v):
    rows, cols = v.shape
    return np.pad(v, ((0, 0), (0, -cols % 128))).reshape(rows, -1, 128)


def scales_of(x, dtype):
    """The smallest power of two under which no value of a row's 128 columns exceeds the type's largest; 1 for zeros."""
    top = np.abs(blocks(x)).max(-1)
    m, e = np.frexp(np.where(top > 0, top, 1.0))
    L, B = np.frexp(LARGEST[dtype])
    p = np.where(m <= L, e - B, e - B + 1)
    return np.where(top > 0, np.exp2(np.maximum(p, -126).astype(np.float64)), 1.0)


def codes_of(x, scales, dtype):
    """x / s, rounded to the nearest code, ties to even, as values."""
    v = x / np.repeat(scales, 128, 1)[:, :x.shape[1]]
    if dtype == torch.int8:
        return np.rint(v)
    mag = np.abs(v)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(mag, 2.0 ** -40))), -6.0) - 3)
    return np.rint(v / step) * step


def values(q, scales):
    """What codes stand for."""
    cols = q.shape[-1]
    q2, s2 = f64(q).reshape(-1, cols), f64(scales).reshape(-1, -(-cols // 128))
    return q2 * np.repeat(s2, 128, 1)[:, :cols]


def weight_gradient(dy, v, w, b):
    """dw, db and their bounds: the matrix cores add 32 rows an instruction, in no fewer than groups of four: a rounding for every
    four rows, and 32 partial sums behind that."""
    rows = dy.shape[0]
    adds = rows / 4 + 48
    G, db = dy.T @ v, dy.sum(0)
    e_G, e_db = adds * U * (np.abs(dy).T @ np.abs(v)), adds * U * np.abs(dy).sum(0)
    dw, e_dw = G, e_G
    if w is not None:
        dw, e_dw = G * w, e_G * np.abs(w) + 2 * U * np.abs(G * w)
    if b is not None:
        rank1 = db[:, None] * b
        dw, e_dw = dw + rank1, e_dw + e_db[:, None] * np.abs(b) + 2 * U * (np.abs(dw) + 2 * np.abs(rank1))
    return (dw, db), (e_dw, e_db)
