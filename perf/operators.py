"""Layer norm, activations kept in 8 bits, and the gradients that are computed from them, as cases that can be timed and compared.

Kinds (`case["kind"]`):

  norm           y = xhat w + b, xhat = (x - mean) rstd, row by row; with `keep`, xhat is also written in 8 bits, as the backward
                 pass will read it, and comes back here as the values that the codes stand for
  norm_backward  the gradients of x, w and b, out of x itself (`keep` "none") or out of xhat in 8 bits
  keep           an activation into 8 bits and back: codes with one power of two as scale for a row's 128 columns
  weights        a linear layer's weight gradient dW = dz^T y and db = the sums of dz, out of activations in 8 bits; with `norm`, what
                 is kept is a layer norm's xhat, and y = xhat w + b is meant
  step           forward and backward of a layer norm and the bf16 linear layer behind it; xhat in 8 bits is all that is kept
                 of the activations

Sizes are those of the benchmark and the tests, and what lies between and beside them: `draw` takes row counts from one
token to a large batch, widths from a head's to a wide layer's, a quarter of them multiples of nothing."""
import math

import torch
import torch.nn.functional as F

own = False

EPS = 1e-5
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


def listed():
    return [
        # one token of one request: latency and launches are all there is
        dict(name="norm_one_token", kind="norm", type="bf16", params="bf16", keep="none", rows=1, cols=7168),
        # the norm of every head of a long prompt: many short rows
        dict(name="norm_heads", kind="norm", type="fp16", params="f32", keep="none", rows=131072, cols=128),
        # a training batch through the norm in front of a wide layer, kept for the backward pass
        dict(name="norm_batch_kept", kind="norm", type="bf16", params="f32", keep="int8", rows=6144, cols=7168),
        # its backward pass where x itself was kept
        dict(name="norm_backward", kind="norm_backward", type="bf16", params="f32", keep="none", rows=8192, cols=4096),
        # and out of 8 bits, on sizes that are multiples of nothing
        dict(name="norm_backward_kept_ragged", kind="norm_backward", type="fp16", params="fp16", keep="fp8", rows=1999, cols=3001),
        # sixteen rows on their way into 8 bits and back: two launches
        dict(name="keep_small", kind="keep", type="bf16", keep="int8", rows=16, cols=2048),
        # the wide inner activation of a large batch
        dict(name="keep_wide", kind="keep", type="bf16", keep="fp8", rows=6144, cols=14336),
        # the gradient of the linear layer behind a norm
        dict(name="weights_behind_norm", kind="weights", type="bf16", out="f32", keep="int8", norm=True, rows=4096, n=4096, cols=2048),
        # ragged in every size: the token count is the contraction's length
        dict(name="weights_ragged", kind="weights", type="fp16", out="f32", keep="fp8", norm=False, rows=1999, n=3001, cols=1000),
        # many tokens against a narrow layer: few tiles of the result, a long contraction
        dict(name="weights_many_tokens", kind="weights", type="bf16", out="f32", keep="int8", norm=False, rows=32768, n=512, cols=1024),
        # the largest product
        dict(name="weights_large", kind="weights", type="bf16", out="bf16", keep="int8", norm=True, rows=8192, n=8192, cols=4096),
        # a training step through both layers
        dict(name="step", kind="step", keep="int8", rows=4096, n=4096, cols=2048),
    ]


# ---------------------------------------------------------------------------------------------------------------------
# more cases of the same ranges
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: a multiple of 128 half of the time, else of 16, 8 or of nothing."""
    unit = rng.choice([128, 128, 128, 128, 16, 8, 1, 1])
    return max(unit, _log_int(rng, lo, hi) // unit * unit)


def _at_most(case, elements=None, flops=None):
    """The case with its rows cut until it costs no more than the largest listed one."""
    while case["rows"] > 1 and (case["rows"] * max(case["cols"], case.get("n", 0)) > elements or
                                (flops and 2.0 * case["rows"] * case["n"] * case["cols"] > flops)):
        case["rows"] = case["rows"] * 5 // 8
    return case


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_backward", "norm_backward", "keep", "weights", "weights", "weights", "step"])
    if kind in ("norm", "norm_backward"):
        t = rng.choice(["bf16", "bf16", "fp16", "f32"])
        return _at_most(dict(kind=kind, type=t, params=rng.choice(["f32", t]), keep=rng.choice(["none", "int8", "fp8"]),
                             rows=_log_int(rng, 1, 65536), cols=_width(rng, 64, 14336)), 4.0e7)
    if kind == "keep":
        return _at_most(dict(kind=kind, type=rng.choice(["bf16", "fp16", "f32"]), keep=rng.choice(["int8", "fp8"]),
                             rows=_log_int(rng, 1, 32768), cols=_width(rng, 64, 14336)), 4.0e7)
    if kind == "weights":
        return _at_most(dict(kind=kind, type=rng.choice(["bf16", "bf16", "fp16"]), out=rng.choice(["f32", "f32", "bf16"]),
                             keep=rng.choice(["int8", "fp8"]), norm=rng.choice([True, False]), rows=_log_int(rng, 64, 32768),
                             n=_width(rng, 256, 8192), cols=_width(rng, 256, 8192)), 8.0e7, 4.0e11)
    return _at_most(dict(kind=kind, keep=rng.choice(["int8", "fp8"]), rows=_log_int(rng, 128, 8192),
                         n=_width(rng, 512, 4096), cols=_width(rng, 512, 4096)), 4.0e7, 6.9e10)


# ---------------------------------------------------------------------------------------------------------------------
def _activations(g, rows, cols):
    """Normally distributed, with channels of different size and rows off centre; the last rows of a batch are padding."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x.mul_(torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda")))
    x.add_(0.3 * torch.randn(rows, 1, generator=g, device="cuda"))
    x[rows - rows // 64:] = 0
    return x


def _gradients(g, rows, cols):
    """What arrives from behind: nothing for padding."""
    dy = torch.randn(rows, cols, generator=g, device="cuda").mul_(cols ** -0.5)
    dy[rows - rows // 64:] = 0
    return dy


def _parameters(g, cols, dtype):
    return ((1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dtype),
            (0.1 * torch.randn(cols, generator=g, device="cuda")).to(dtype))


def _statistics(x):
    mean = x.mean(-1)
    return mean, torch.rsqrt((x - mean[:, None]).square().mean(-1) + EPS)


def _blocks(x):
    rows, cols = x.shape
    return F.pad(x, (0, -cols % 128)).view(rows, -1, 128)


def _encode(x, keep):
    """Codes, and for every 128 columns of a row the smallest power of two with which no value exceeds the type's largest
    number, 127 or 448; 1 for zeros."""
    b = _blocks(x)
    m, e = torch.frexp(b.abs().amax(-1))
    p = torch.where(m <= 127 / 128, e - 7, e - 6) if keep == "int8" else torch.where(m <= 448 / 512, e - 9, e - 8)
    p = torch.where(m == 0, 0, p)
    one = torch.ones((), device=x.device)
    v = (b * torch.ldexp(one, -p)[..., None]).flatten(1)[:, :x.shape[1]]
    return (torch.round(v).to(torch.int8) if keep == "int8" else v.to(torch.float8_e4m3fn)), torch.ldexp(one, p)


def _decode(q, scales):
    return (_blocks(q.float()) * scales[..., None]).flatten(1)[:, :q.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, rows, cols = case["kind"], case["rows"], case["cols"]
    state = dict(case, params=_TYPES.get(case.get("params")))
    if kind == "keep":
        return dict(state, x=_activations(g, rows, cols).to(_TYPES[case["type"]]))
    if kind in ("norm", "norm_backward"):
        dtype = _TYPES[case["type"]]
        state["x"] = x = _activations(g, rows, cols).to(dtype)
        state["w"], state["b"] = _parameters(g, cols, state["params"])
        if kind == "norm_backward":
            state["mean"], state["rstd"] = _statistics(x.float())
            state["dy"] = _gradients(g, rows, cols).to(dtype)
            if case["keep"] != "none":
                xhat = (x.float() - state["mean"][:, None]) * state["rstd"][:, None]
                state["q"], state["scales"] = _encode(xhat, case["keep"])
                del state["x"]
        return state
    n, dtype = case["n"], _TYPES[case.get("type", "bf16")]
    state["dz"] = _gradients(g, rows, n).to(dtype)
    if kind == "weights":
        x = _activations(g, rows, cols)
        state["w"] = state["b"] = None
        if case["norm"]:
            mean, rstd = _statistics(x)
            x = (x - mean[:, None]) * rstd[:, None]
            state["w"], state["b"] = _parameters(g, cols, dtype)
        state["q"], state["scales"] = _encode(x, case["keep"])
        return state
    state["x"] = _activations(g, rows, cols).to(dtype)
    state["w"], state["b"] = _parameters(g, cols, dtype)
    state["W"] = torch.randn(n, cols, generator=g, device="cuda").mul_(cols ** -0.5).to(dtype)
    return state


# ---------------------------------------------------------------------------------------------------------------------
# the plain form: 32 bits, rounded once at the end
def _norm(s):
    x = s["x"].float()
    mean, rstd = _statistics(x)
    xhat = (x - mean[:, None]) * rstd[:, None]
    return xhat, mean, rstd, xhat * s["w"].float() + s["b"].float()


def _norm_gradients(dy, xhat, rstd, w):
    g = dy * w.float()
    dx = rstd[:, None] * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx, (dy * xhat).sum(0), dy.sum(0)


def _weight_gradients(dz, y, w, b):
    if w is not None:
        y = y * w.float() + b.float()
    return dz.t() @ y, dz.sum(0)


def _plain(s):
    kind = s["kind"]
    if kind == "norm":
        xhat, mean, rstd, y = _norm(s)
        out = dict(y=y.to(s["x"].dtype), mean=mean, rstd=rstd)
        return out if s["keep"] == "none" else dict(out, kept=_decode(*_encode(xhat, s["keep"])).bfloat16())
    if kind == "norm_backward":
        xhat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None] if s["keep"] == "none" else _decode(s["q"], s["scales"])
        dx, dw, db = _norm_gradients(s["dy"].float(), xhat, s["rstd"], s["w"])
        return dict(dx=dx.to(s["dy"].dtype), dw=dw.to(s["params"]), db=db.to(s["params"]))
    if kind == "keep":
        return _decode(*_encode(s["x"].float(), s["keep"])).to(s["x"].dtype)
    if kind == "weights":
        dW, db = _weight_gradients(s["dz"].float(), _decode(s["q"], s["scales"]), s["w"], s["b"])
        return dict(dW=dW.to(_TYPES[s["out"]]), db=db)
    xhat, _, rstd, y = _norm(s)
    W, dz, kept = s["W"].float(), s["dz"].float(), _decode(*_encode(xhat, s["keep"]))
    dW, dbias = _weight_gradients(dz, kept, s["w"], s["b"])
    dx, dw, db = _norm_gradients(dz @ W, kept, rstd, s["w"])
    half = dict(z=y @ W.t(), dx=dx, dW=dW, dw=dw, db=db)
    return dict({k: v.bfloat16() for k, v in half.items()}, dbias=dbias)


# ---------------------------------------------------------------------------------------------------------------------
# the same through the library
def _through_library(s):
    import qgemm_amd as Q

    kind, keep = s["kind"], s["keep"]
    if kind == "norm":
        if keep == "none":
            y, mean, rstd = Q.layer_norm(s["x"], s["w"], s["b"], EPS)
            return dict(y=y, mean=mean, rstd=rstd)
        y, mean, rstd, q, scales = Q.layer_norm(s["x"], s["w"], s["b"], EPS, keep=_TYPES[keep])
        return dict(y=y, mean=mean, rstd=rstd, kept=Q.restore(q, scales, torch.bfloat16))
    if kind == "norm_backward":
        if keep == "none":
            dx, dw, db = Q.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["w"])
        else:
            dx, dw, db = Q.layer_norm_backward(s["dy"], s["q"], None, s["rstd"], s["w"], scales=s["scales"])
        return dict(dx=dx, dw=dw, db=db)
    if kind == "keep":
        return Q.restore(*Q.checkpoint(s["x"], _TYPES[keep]), s["x"].dtype)
    if kind == "weights":
        dW, db = Q.weight_gradient(s["dz"], s["q"], s["scales"], s["w"], s["b"], out_dtype=_TYPES[s["out"]])
        return dict(dW=dW, db=db)
    x, w, W, dz = s["x"], s["w"], s["W"], s["dz"]
    y, _, rstd, q, scales = Q.layer_norm(x, w, s["b"], EPS, keep=_TYPES[keep])
    z = Q.gemm(y, W, torch.empty_like(dz), "nk")
    dW, dbias = Q.weight_gradient(dz, q, scales, w, s["b"], out_dtype=torch.bfloat16)
    dy = Q.gemm(dz, W, torch.empty(x.shape, dtype=torch.float32, device=x.device), "kn")
    dx, dw, db = Q.layer_norm_backward(dy, q, None, rstd, w, scales=scales, out_dtype=x.dtype)
    return dict(z=z, dx=dx, dW=dW, dw=dw, db=db, dbias=dbias)


def run(state):
    return _through_library(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    """Every input read once, every output written once; what passes between two calls is not counted, nor are the codes of an
    activation that comes back within the pass."""
    kind, rows, cols, n = case["kind"], case["rows"], case["cols"], case.get("n", 0)
    size = lambda t: _TYPES[t].itemsize  # noqa: E731
    params, codes = 2 * cols * size(case.get("params") or "bf16"), rows * (cols + 4 * -(-cols // 128))
    if kind == "norm":
        return {"bytes": rows * (cols * (2 * size(case["type"]) + (2 if case["keep"] != "none" else 0)) + 8) + params, "flops": 8.0 * rows * cols}
    if kind == "norm_backward":
        kept = rows * (cols * size(case["type"]) + 4) if case["keep"] == "none" else codes
        return {"bytes": rows * (2 * cols * size(case["type"]) + 4) + kept + params * 3 // 2, "flops": 12.0 * rows * cols}
    if kind == "keep":
        return {"bytes": 2 * rows * cols * size(case["type"]), "flops": 4.0 * rows * cols}
    if kind == "weights":
        return {"bytes": 2 * rows * n + codes + (4 * cols if case["norm"] else 0) + n * cols * size(case["out"]) + 4 * n, "flops": 2.0 * rows * n * cols}
    return {"bytes": 2 * (2 * rows * cols + 2 * rows * n + 2 * n * cols + 4 * cols) + 4 * n, "flops": 6.0 * rows * n * cols}


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions
def _exact_moments(x):
    n = x.shape[1]
    centre = x.sum(1, keepdim=True) / n
    away = x - centre
    return centre.squeeze(1), 1 / ((away * away).sum(1) / n + EPS).sqrt(), away


def _exact_values(codes, scales):
    return codes.double() * scales.double().repeat_interleave(128, 1)[:, :codes.shape[1]]


def _exact_rounded(x, keep):
    """x in 8 bits, as values: a power of two for each 128 columns, from its definition."""
    rows, cols = x.shape
    largest = 127.0 if keep == "int8" else 448.0
    top = F.pad(x.abs(), (0, -cols % 128)).view(rows, -1, 128).amax(2)
    unit = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, largest) / largest)))
    unit = torch.where(unit * largest < top, 2 * unit, unit)
    unit = torch.where(unit / 2 * largest >= torch.where(top > 0, top, 2 * largest), unit / 2, unit)
    unit = unit.repeat_interleave(128, 1)[:, :cols]
    v = x / unit
    if keep == "int8":
        return torch.round(v) * unit
    # three bits behind the leading one, multiples of 2^-9 at the least
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -40))), min=-6.0) - 3)
    return torch.round(v / step) * step * unit


def _exact_norm_gradients(dy, xhat, rstd, w):
    n = dy.shape[1]
    g = dy * w
    a, b = g.sum(1, keepdim=True) / n, (g * xhat).sum(1, keepdim=True) / n
    return (g - a - xhat * b) * rstd[:, None], (dy * xhat).sum(0), dy.sum(0)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "keep":
        return _exact_rounded(s["x"].double(), case["keep"])
    w, b = (None if s[k] is None else s[k].double() for k in ("w", "b"))
    if kind == "norm":
        mean, rstd, away = _exact_moments(s["x"].double())
        xhat = away * rstd[:, None]
        out = dict(y=xhat * w + b, mean=mean, rstd=rstd)
        # (what is kept is measured against xhat itself: rounding is part of its error)
        return out if case["keep"] == "none" else dict(out, kept=xhat)
    if kind == "norm_backward":
        rstd = s["rstd"].double()
        xhat = (s["x"].double() - s["mean"].double()[:, None]) * rstd[:, None] if case["keep"] == "none" else _exact_values(s["q"], s["scales"])
        dx, dw, db = _exact_norm_gradients(s["dy"].double(), xhat, rstd, w)
        return dict(dx=dx, dw=dw, db=db)
    dz = s["dz"].double()
    if kind == "weights":
        y = _exact_values(s["q"], s["scales"])
        if w is not None:
            y = y * w + b
        return dict(dW=torch.mm(dz.t().contiguous(), y), db=dz.sum(0))
    W = s["W"].double()
    _, rstd, away = _exact_moments(s["x"].double())
    xhat = away * rstd[:, None]
    kept = _exact_rounded(xhat, case["keep"])
    dx, dw, db = _exact_norm_gradients(torch.mm(dz, W), kept, rstd, w)
    return dict(z=torch.mm(xhat * w + b, W.t().contiguous()), dx=dx, dW=torch.mm(dz.t().contiguous(), kept * w + b), dw=dw, db=db, dbias=dz.sum(0))
