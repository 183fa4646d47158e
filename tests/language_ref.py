"""Root-mean-square norm, adapters and log probabilities in 64 bits, from the formulas, with the error that fp32 sums may leave (u = 2^-24 is
half a last place of fp32; see training_ref for bounds on what is stored)."""
import numpy as np

from tests.training_ref import U, blocks

EPS = 1e-6


def rms(h, w, eps):
    """y, rstd and their bounds.  A square passes through no more than 44 roundings on its way into the row's sum (an octet's sum, up to eight octets of a
    lane one after the other, ten exchanges), and one for every 2048 columns in rows that no registers hold; squares are positive, so that is
    relative to the sum, and half of it to rstd."""
    n = h.shape[-1]
    rstd = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    rel = 0.5 * (46 + n / 2048) * U + 4 * U
    y = h * rstd * (1.0 if w is None else w)
    return (y, rstd), (np.abs(y) * (rel + 3 * U), rstd * rel)


def rms_gradients(dy, h, rstd, w, dh):
    """dx, dw and their bounds; rstd as it was handed over."""
    rows, n = dy.shape
    g, xhat = dy if w is None else dy * w, h * rstd
    b = (g * xhat).mean(-1, keepdims=True)
    e_b = (48 + n / 2048) * U * np.abs(g * xhat).mean(-1, keepdims=True)
    dx = rstd * (g - xhat * b)
    e_dx = rstd * (U * np.abs(g) + np.abs(xhat) * e_b + 4 * U * (np.abs(g) + np.abs(xhat * b))) + U * np.abs(dx)
    if dh is not None:
        dx = dx + dh
        e_dx = e_dx + U * np.abs(dx)
    adds = rows / 16 + 80                            # (no more than a sixteenth of the rows one after the other, 64 partial sums behind that)
    return (dx, (dy * xhat).sum(0)), (e_dx, (adds + 2) * U * np.abs(dy * xhat).sum(0))


def check_codes(q, scales, y, e_y, largest, stored):
    """Codes and scales (as numbers) of y, which is known to e_y: s = max|y| / largest, |q s - y| half a step."""
    top, slack = np.abs(blocks(y)).max(-1), np.abs(blocks(e_y)).max(-1)
    want = np.where(top > 0, top / largest, 1.0)
    assert (np.abs(scales - want) <= slack / largest + 2 * U * want + (top <= slack)).all()
    full = np.repeat(scales, 128, 1)[:, :y.shape[1]]
    half = full / 2 if stored == "int8" else np.maximum(np.abs(y) * 2.0 ** -4, full * 2.0 ** -10)
    assert (np.abs(q * full - y) <= half * (1 + 4 * U) + 2 * e_y + 4 * U * np.abs(y)).all()
    assert np.abs(q).max() <= largest


# The matrix cores add 32 products an instruction, in no fewer than groups of four: a rounding for every four terms, and up to 80 behind that (splits of
# the sum, four waves, an accumulator that y starts).
def _adds(n):
    return n / 4 + 80


def adapters(y, x, A, B, ids, s, parts):
    """out, u and their bounds: u is fp32 and goes on in 2 or 3 bf16 parts, each of which leaves 2^-9 of what it was split off."""
    out, e_out = y.copy(), U * np.abs(y)
    u, e_u = np.zeros((len(x), A.shape[1])), np.zeros((len(x), A.shape[1]))
    for i in range(len(A)):
        rows = np.nonzero(ids == i)[0]
        if not len(rows):
            continue
        u[rows] = x[rows] @ A[i].T
        e_u[rows] = _adds(A.shape[2]) * U * (np.abs(x[rows]) @ np.abs(A[i]).T)
        out[rows] += s[i] * (u[rows] @ B[i])
        size = s[i] * (np.abs(u[rows]) @ np.abs(B[i]))
        e_out[rows] = s[i] * (e_u[rows] @ np.abs(B[i])) + (2.0 ** (-9 * parts) + (2 * parts * _adds(A.shape[1])) * U) * (size + np.abs(y[rows])) + U * np.abs(out[rows])
    return (out, u), (e_out, e_u)


def adapter_gradients(dy, x, u, A, B, ids, s, dx, parts, grad_parts):
    out = adapters(dx, dy, B, A, ids, s, parts)
    v, e_v = out[0][1], out[1][1]
    dA, dB, e_dA, e_dB = (np.zeros(t.shape) for t in (A, B, A, B))
    for i in range(len(A)):
        rows = np.nonzero(ids == i)[0]
        if not len(rows):
            continue
        rel = 2.0 ** (-9 * grad_parts) + 2 * grad_parts * _adds(len(rows)) * U
        for to, e_to, r, e_r, z in ((dA, e_dA, v, e_v, x), (dB, e_dB, u, None, dy)):
            to[i] = s[i] * (r[rows].T @ z[rows])
            e_to[i] = s[i] * rel * (np.abs(r[rows]).T @ np.abs(z[rows]))
            if e_r is not None:
                e_to[i] += s[i] * (e_r[rows].T @ np.abs(z[rows]))
    return (out[0][0], dA, dB), (out[1][0], e_dA, e_dB)


def log_probabilities(x):
    """log p, entropy, lse and their bounds.  An exponential's argument is rounded twice and its value by a last place; a thread adds up to eight of each octet one
    after the other and puts its sums right, by another such exponential, no more than once an octet; 20 exchanges behind that."""
    m = x.max(-1, keepdims=True)
    empty = np.isneginf(m)
    d = x - np.where(empty, 0.0, m)
    e = np.exp(d)
    S = np.where(empty, 1.0, e.sum(-1, keepdims=True))
    p, dd = e / S, np.where(e > 0, d, 0.0)
    lse = np.where(empty, -np.inf, m + np.log(S))
    with np.errstate(invalid="ignore"):
        lp = np.where(np.isneginf(x), -np.inf, x - np.where(empty, 0.0, lse))
    T = (p * dd).sum(-1, keepdims=True)
    H = np.where(empty, 0.0, np.log(S) - T)
    octets = x.shape[-1] / 2048 + 2
    each = U * (2 * np.abs(dd) + 4) + U * (10 * octets + 40 + 4 * np.abs(dd).max(-1, keepdims=True) * (e > 0))
    e_s = (p * each).sum(-1, keepdims=True)
    e_lse = e_s + 3 * U * (np.abs(np.log(S)) + np.abs(np.where(empty, 0.0, lse)) + np.abs(np.where(empty, 0.0, m)))
    e_H = e_s * (1 + np.abs(T)) + (p * np.abs(dd) * each).sum(-1, keepdims=True) + 4 * U * (np.log(S) + np.abs(T))
    with np.errstate(invalid="ignore"):
        e_lp = e_lse + U * np.where(np.isfinite(lp), np.abs(lp) + np.abs(np.where(np.isfinite(x), x, 0.0)), 0.0)
    return (lp, H[..., 0], lse[..., 0]), (e_lp, e_H[..., 0], e_lse[..., 0])


def logit_gradients(x, tokens, lse, H, a, b):
    """dlogits and its bound; lse and H as they were handed over."""
    rows = np.arange(len(x))
    none = np.isneginf(lse)[:, None]
    safe = np.where(none, 0.0, lse[:, None])
    lp = np.where(none | np.isneginf(x), -np.inf, x - safe)
    p, l = np.exp(lp), np.where(np.isneginf(lp), 0.0, lp)
    asked = (tokens >= 0) & (tokens < x.shape[1]) & ~none[:, 0]
    a = np.where(asked, a, 0.0)[:, None]
    b = b[:, None]
    H = H[:, None]
    inner = a + b * (l + H)
    dx = -p * inner
    dx[rows[asked], tokens[asked]] += a[asked, 0]
    finite = np.where(np.isfinite(x), np.abs(x), 0.0)
    e_l = U * (np.abs(l) + finite)
    e = p * (np.abs(inner) * (4 * U + e_l + 2 * U * np.abs(l)) + 4 * U * (np.abs(a) + np.abs(b) * (np.abs(l) + np.abs(H))) + np.abs(b) * e_l) + 2 * U * np.abs(dx)
    e[rows[asked], tokens[asked]] += 2 * U * np.abs(a[asked, 0])
    return dx, e
