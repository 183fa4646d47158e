"""What stands beside the products of a language model, as cases that can be timed and compared: the root-mean-square norm in front of them, low-rank
adapters added to what they give, and the log probabilities read from the last one; each with its gradients.

Kinds (`case["kind"]`):

  norm               h = x + residual, y = h rstd w, row by row; with `codes`, y is also (or only) written in 8 bits with a scale for a row's
                     128 columns, as the block-scaled products read it, and comes back here as the values that the codes stand for
  norm_backward      the gradients of x and w out of h, with the gradient that arrives along the residual stream
  adapters           y + s_i (x A_i^T) B_i where every row has an adapter i of its own, or none
  adapters_backward  the gradients of x, A and B
  log_probabilities  of given tokens, with the entropy and the `top` most probable tokens, out of logits
  logits_backward    the gradient of logits out of those of the log probabilities and entropies

Sizes are those of the benchmark and the tests, generic vocabularies of a power of two and ragged ones, and what lies between: `draw` takes row counts from one token
to a large batch, a part of all widths multiples of nothing."""
import math

import torch
import torch.nn.functional as F

own = False

EPS = 1e-6
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
_LARGEST = {"int8": 127.0, "fp8": 448.0}


def listed():
    return [
        # one token of one request, straight into the operand of an 8-bit product: latency and launches are all there is
        dict(name="norm_one_token", kind="norm", type="bf16", params="bf16", residual=True, codes="fp8", y=False, rows=1, cols=7168),
        # a training batch in front of an 8-bit product, with y itself for the adapters beside that product
        dict(name="norm_batch", kind="norm", type="bf16", params="f32", residual=True, codes="int8", y=True, rows=6144, cols=7168),
        # its backward pass, with what arrives along the residual stream
        dict(name="norm_backward", kind="norm_backward", type="bf16", params="f32", residual=True, rows=8192, cols=4096),
        # and on sizes that are multiples of nothing
        dict(name="norm_backward_ragged", kind="norm_backward", type="fp16", params="fp16", residual=False, rows=1999, cols=3001),
        # a decoding step: a token of each request, most requests with an adapter of their own
        dict(name="adapters_decode", kind="adapters", type="bf16", y_type="bf16", rows=64, adapters=48, rank=16, k=4096, n=4096),
        # prompts of several requests side by side
        dict(name="adapters_prompts", kind="adapters", type="bf16", y_type="bf16", rows=8192, adapters=8, rank=32, k=4096, n=4096),
        # ragged in every size, beside a product that leaves fp32
        dict(name="adapters_ragged", kind="adapters", type="fp16", y_type="f32", rows=1999, adapters=5, rank=12, k=1000, n=3001),
        # many adapters trained at once
        dict(name="adapters_backward", kind="adapters_backward", type="bf16", y_type="bf16", rows=4096, adapters=16, rank=16, k=2048, n=8192),
        # the answer of a decoding step: few rows of a large vocabulary, with twenty alternatives
        dict(name="answers", kind="log_probabilities", type="f32", rows=8, vocabulary=131072, top=20, masked=False),
        # prompts scored: many rows, a part of the vocabulary masked, five alternatives
        dict(name="scores", kind="log_probabilities", type="bf16", rows=2048, vocabulary=65536, top=5, masked=True),
        # a small vocabulary of no round size
        dict(name="scores_small", kind="log_probabilities", type="fp16", rows=77, vocabulary=5003, top=0, masked=True),
        # the backward pass of a policy's update: log probabilities and entropies both have gradients
        dict(name="logits_backward", kind="logits_backward", type="bf16", rows=2048, vocabulary=65536, masked=False),
    ]


# ---------------------------------------------------------------------------------------------------------------------
# more cases of the same ranges
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: a multiple of 128 half of the time, else of 16, 8 or of nothing."""
    unit = rng.choice([128, 128, 128, 128, 16, 8, 1, 1])
    return max(unit, _log_int(rng, lo, hi) // unit * unit)


def _fewer_rows(case, most):
    """The case with its rows cut until `most`, elements or products by row, holds."""
    while case["rows"] > 1 and most(case) > 1:
        case["rows"] = case["rows"] * 5 // 8
    return case


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_backward", "adapters", "adapters", "adapters", "adapters_backward", "log_probabilities", "log_probabilities",
                       "logits_backward"])
    t = rng.choice(["bf16", "bf16", "fp16", "f32"])
    if kind.startswith("norm"):
        case = dict(kind=kind, type=t, params=rng.choice(["f32", t]), residual=rng.random() < 0.7, rows=_log_int(rng, 1, 32768), cols=_width(rng, 64, 14336))
        if kind == "norm":
            case["codes"] = rng.choice(["none", "int8", "fp8"])
            case["y"] = case["codes"] == "none" or rng.random() < 0.5
        return _fewer_rows(case, lambda c: c["rows"] * c["cols"] / 3.3e7)
    if kind.startswith("adapters"):
        case = dict(kind=kind, type=rng.choice(["bf16", "bf16", "fp16"]), rows=_log_int(rng, 1, 8192), adapters=_log_int(rng, 1, 128),
                    rank=rng.choice([4, 8, 8, 16, 16, 16, 32, 32, 64, 128, rng.randint(1, 128)]), k=_width(rng, 256, 8192), n=_width(rng, 256, 8192))
        case["adapters"] = max(1, min(case["adapters"], 2048 // case["rank"]))
        case["y_type"] = rng.choice([case["type"], case["type"], "f32"])
        return _fewer_rows(case, lambda c: c["rows"] * (c["k"] + c["n"]) * max(1, c["rank"] * c["adapters"] / 256) / 6.7e7)
    case = dict(kind=kind, type=t, rows=_log_int(rng, 1, 4096), vocabulary=_log_int(rng, 500, 262144), masked=rng.random() < 0.5)
    if rng.random() < 0.5:
        case["vocabulary"] = max(512, case["vocabulary"] // 512 * 512)
    if kind == "log_probabilities":
        case["top"] = rng.choice([0, 0, 1, 5, 20, 32])
    return _fewer_rows(case, lambda c: c["rows"] * c["vocabulary"] / (6.7e7 if t == "f32" else 1.3e8))


# ---------------------------------------------------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, cols):
    """Normally distributed, with channels of different size; the last rows of a batch are padding."""
    x = _randn(g, rows, cols).mul_(torch.exp(0.5 * _randn(g, cols)))
    x[rows - rows // 64:] = 0
    return x


def _ids(g, rows, adapters):
    """Up to 256 rows are tokens of as many requests; more are prompts, one behind the other.  One request in eight has no adapter."""
    requests = rows if rows <= 256 else max(8, rows // 256)
    of = torch.randint(0, adapters, (requests,), generator=g, device="cuda")
    of = torch.where(torch.rand(requests, generator=g, device="cuda") < 0.125, -1, of)
    if requests == rows:
        return of.int()
    ends = torch.sort(torch.randint(0, rows, (requests - 1,), generator=g, device="cuda")).values
    return of[torch.searchsorted(ends, torch.arange(rows, device="cuda"), right=True)].int()


def _logits(g, case):
    """A few tokens far above the rest; masked: half of the vocabulary at minus infinity or the type's lowest value, and now and then a row with
    nothing left."""
    rows, v, dtype = case["rows"], case["vocabulary"], _TYPES[case["type"]]
    x = torch.empty(rows, v, dtype=dtype, device="cuda")
    x.normal_(0, 2.0, generator=g)
    x.scatter_add_(1, torch.randint(0, v, (rows, 16), generator=g, device="cuda"), (8 * torch.rand(rows, 16, generator=g, device="cuda")).to(dtype))
    if case["masked"]:
        out = torch.rand(v, generator=g, device="cuda") < 0.5
        x[0::3, out] = float("-inf")
        x[1::3, out] = torch.finfo(dtype).min
        x[5::67] = float("-inf")
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, rows = case["kind"], case["rows"]
    dtype, state = _TYPES[case["type"]], dict(case)
    if kind.startswith("norm"):
        cols = case["cols"]
        state["w"] = (1 + 0.2 * _randn(g, cols)).to(_TYPES[case["params"]])
        if kind == "norm":
            state["x"] = _activations(g, rows, cols).to(dtype)
            state["residual"] = _randn(g, rows, cols).mul_(2).to(dtype) if case["residual"] else None
            return state
        state["h"] = h = _activations(g, rows, cols).to(dtype)
        state["rstd"] = torch.rsqrt(h.float().square().mean(-1) + EPS)
        state["dy"] = _randn(g, rows, cols).mul_(cols ** -0.5).to(dtype)
        state["dh"] = _randn(g, rows, cols).mul_(cols ** -0.5).to(dtype) if case["residual"] else None
        return state
    if kind.startswith("adapters"):
        a, r, k, n, y_type = case["adapters"], case["rank"], case["k"], case["n"], _TYPES[case["y_type"]]
        state["ids"] = _ids(g, rows, a)
        state["x"] = _activations(g, rows, k).to(dtype)
        state["A"], state["B"] = _randn(g, a, r, k).mul_(k ** -0.5).to(dtype), _randn(g, a, r, n).mul_(0.3 * r ** -0.5).to(dtype)
        state["scaling"] = 0.5 + torch.rand(a, generator=g, device="cuda")
        if kind == "adapters":
            state["y"] = _randn(g, rows, n).to(y_type)
            return state
        state["dy"], state["dx"] = _randn(g, rows, n).mul_(n ** -0.5).to(dtype), _randn(g, rows, k).mul_(n ** -0.5).to(y_type)
        state["u"] = _own_rank(state["x"].float() @ state["A"].float().flatten(0, 1).t(), state["ids"], a)
        return state
    state["logits"] = _logits(g, case)
    tokens = torch.randint(0, case["vocabulary"], (rows, 1), generator=g, device="cuda")
    asked = state["logits"].gather(1, tokens)                      # (no one asks for what the lowest value masks; minus infinity may come up)
    lowest = asked == torch.finfo(dtype).min
    state["tokens"] = torch.where(lowest, state["logits"].argmax(1, keepdim=True), tokens)[:, 0]
    state["tokens"][7::64] = -100                                  # padding: nothing is asked
    if kind == "logits_backward":
        _, state["entropy"], state["lse"] = _statistics(state["logits"].float())
        state["dlogp"], state["dentropy"] = _randn(g, rows).div_(rows), _randn(g, rows).div_(100 * rows)
    return state


# ---------------------------------------------------------------------------------------------------------------------
# the plain form: 32 bits, rounded once at the end
def _blocks(x):
    return F.pad(x, (0, -x.shape[1] % 128)).unflatten(1, (-1, 128))


def _through_codes(y, codes):
    """y in 8 bits with a scale for every 128 columns of a row, as values."""
    b = _blocks(y)
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, top / _LARGEST[codes], 1.0)
    v = (b / scale).clamp(-_LARGEST[codes], _LARGEST[codes])
    q = torch.round(v) if codes == "int8" else v.to(torch.float8_e4m3fn).float()
    return (q * scale).flatten(1)[:, :y.shape[1]].bfloat16()


def _own_rank(every, ids, adapters):
    """[rows, adapters x rank] to the rank of each row's own adapter; zeros where it has none."""
    every = every.unflatten(1, (adapters, -1))
    own_one = every[torch.arange(len(ids), device=ids.device), ids.clamp(min=0).long()]
    return torch.where((ids >= 0)[:, None], own_one, 0.0)


def _at_own(u, ids, adapters):
    """[rows, rank] to [rows, adapters x rank]: zeros but at the row's own adapter."""
    return (F.one_hot((ids + 1).long(), adapters + 1)[:, 1:, None] * u[:, None, :]).flatten(1)


def _plain_adapters(s):
    ids, a = s["ids"], s["adapters"]
    A, B, x = s["A"].float().flatten(0, 1), s["B"].float().flatten(0, 1), s["x"].float()
    scaling = s["scaling"][ids.clamp(min=0).long()][:, None]
    if s["kind"] == "adapters":
        u = _own_rank(x @ A.t(), ids, a)
        return (s["y"].float() + _at_own(u * scaling, ids, a) @ B).to(s["y"].dtype)
    dy = s["dy"].float()
    v = _at_own(_own_rank(dy @ B.t(), ids, a) * scaling, ids, a)
    dx = (s["dx"].float() + v @ A).to(s["dx"].dtype)
    return dict(dx=dx, dA=(v.t() @ x).view(s["A"].shape), dB=(_at_own(s["u"] * scaling, ids, a).t() @ dy).view(s["B"].shape))


def _statistics(x):
    """x - max, entropy, logarithm of the exponentials' sum; a row with nothing but minus infinity has no entropy."""
    m = x.amax(-1, keepdim=True)
    d = x - torch.where(m == float("-inf"), 0.0, m)
    e = torch.exp(d)
    s = e.sum(-1)
    h = torch.where(s > 0, torch.log(s) - torch.where(e > 0, e * d, 0.0).sum(-1) / s, 0.0)
    return d, h, torch.where(s > 0, m[:, 0] + torch.log(s), float("-inf"))


def _of_tokens(x, lse, tokens):
    """A token that is none has the logarithm 0."""
    asked = x.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    return torch.where(tokens < 0, 0.0, torch.where(lse == float("-inf"), lse, asked - lse))


def _top(x, k):
    """The k largest of each row, the lowest index first where they are equal: numbers that order as the values do, and the index, in 64 bits."""
    i = (x + 0.0).view(torch.int32).long()
    key = torch.where(i < 0, -2 ** 31 - 1 - i, i) * 2 ** 32 + (2 ** 31 - torch.arange(x.shape[1], device=x.device))
    index = torch.topk(key, k, dim=1).indices
    return x.gather(1, index), index


def _plain_logits(s):
    x, tokens = s["logits"].float(), s["tokens"]
    if s["kind"] == "log_probabilities":
        _, h, lse = _statistics(x)
        out = dict(logp=_of_tokens(x, lse, tokens), entropy=h, lse=lse)
        if s["top"]:
            values, out["indices"] = _top(x, s["top"])
            out["values"] = torch.where(values == float("-inf"), values, values - lse[:, None])
        return out
    lp = torch.where(s["lse"][:, None] == float("-inf"), float("-inf"), x - s["lse"][:, None])
    p = torch.exp(lp)
    a = torch.where(tokens < 0, 0.0, s["dlogp"])[:, None]
    dx = -p * a - torch.where(p > 0, p * (lp + s["entropy"][:, None]), 0.0) * s["dentropy"][:, None]
    dx.scatter_add_(1, tokens.clamp(min=0)[:, None], torch.where(s["lse"][:, None] == float("-inf"), 0.0, a))
    return dx.to(s["logits"].dtype)


def _plain(s):
    kind = s["kind"]
    if kind == "norm":
        h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)
        rstd = torch.rsqrt(h.float().square().mean(-1) + EPS)
        y = h.float() * rstd[:, None] * s["w"].float()
        out = dict(rstd=rstd, h=h) if s["residual"] is not None else dict(rstd=rstd)
        if s["y"]:
            out["y"] = y.to(s["x"].dtype)
        if s["codes"] != "none":
            out["quantized"] = _through_codes(y, s["codes"])
        return out
    if kind == "norm_backward":
        dy, xhat, rstd = s["dy"].float(), s["h"].float() * s["rstd"][:, None], s["rstd"][:, None]
        g = dy * s["w"].float()
        dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
        return dict(dx=(dx if s["dh"] is None else dx + s["dh"].float()).to(s["dy"].dtype), dw=(dy * xhat).sum(0).to(s["w"].dtype))
    return _plain_adapters(s) if kind.startswith("adapters") else _plain_logits(s)


# ---------------------------------------------------------------------------------------------------------------------
# the same through the library
def _through_library(s):
    import qgemm_amd as Q

    kind = s["kind"]
    if kind == "norm":
        codes = None if s["codes"] == "none" else _TYPES[s["codes"]]
        y, h, rstd, *quantized = Q.rms_norm(s["x"], s["w"], EPS, residual=s["residual"], codes=codes, store_y=s["y"])
        out = dict(rstd=rstd, h=h) if s["residual"] is not None else dict(rstd=rstd)
        if s["y"]:
            out["y"] = y
        if quantized:
            out["quantized"] = Q.restore(*quantized, torch.bfloat16)
        return out
    if kind == "norm_backward":
        dx, dw = Q.rms_norm_backward(s["dy"], s["h"], s["rstd"], s["w"], dh=s["dh"])
        return dict(dx=dx, dw=dw)
    if kind == "adapters":
        return Q.add_adapters(s["y"], s["x"], s["A"], s["B"], Q.group_rows(s["ids"], s["adapters"]), s["scaling"])
    if kind == "adapters_backward":
        groups = Q.group_rows(s["ids"], s["adapters"])
        dx, dA, dB = Q.add_adapters_backward(s["dy"], s["x"], s["u"], s["A"], s["B"], groups, s["scaling"], dx=s["dx"])
        return dict(dx=dx, dA=dA, dB=dB)
    if kind == "log_probabilities":
        logp, entropy, lse, *top = Q.log_probabilities(s["logits"], s["tokens"], top=s["top"])
        out = dict(logp=logp, entropy=entropy, lse=lse)
        return dict(out, values=top[0], indices=top[1]) if top else out
    return Q.log_probabilities_backward(s["logits"], s["tokens"], s["lse"], s["entropy"], s["dlogp"], s["dentropy"])


def run(state):
    return _through_library(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    """Every input read once, every output written once; the codes of a norm are counted as codes, not as what comes back of them."""
    kind, rows, size = case["kind"], case["rows"], _TYPES[case["type"]].itemsize
    if kind == "norm":
        cols = case["cols"]
        codes = rows * (cols + 4 * -(-cols // 128)) if case["codes"] != "none" else 0
        moved = rows * cols * size * (1 + (2 if case["residual"] else 0) + (1 if case["y"] else 0)) + codes + 4 * rows
        return {"bytes": moved + cols * _TYPES[case["params"]].itemsize, "flops": 6.0 * rows * cols}
    if kind == "norm_backward":
        cols = case["cols"]
        return {"bytes": rows * (cols * size * (4 if case["residual"] else 3) + 4) + 2 * cols * _TYPES[case["params"]].itemsize, "flops": 10.0 * rows * cols}
    if kind.startswith("adapters"):
        a, r, k, n, y = case["adapters"], case["rank"], case["k"], case["n"], _TYPES[case["y_type"]].itemsize
        used = a * (1 - (1 - 1 / a) ** (rows if rows <= 256 else max(8, rows // 256)))          # adapters that any request has
        if kind == "adapters":
            return {"bytes": int(rows * (k * size + 2 * n * y + 4) + used * r * (k + n) * size), "flops": 2.0 * rows * r * (k + n)}
        return {"bytes": int(rows * ((k + n) * size + 2 * k * y + 4 * r + 4) + used * r * (k + n) * size + a * r * (k + n) * 4), "flops": 4.0 * rows * r * (k + n)}
    v = case["vocabulary"]
    if kind == "log_probabilities":
        return {"bytes": rows * (v * size + 20 + 12 * case["top"]), "flops": 6.0 * rows * v}
    return {"bytes": rows * (2 * v * size + 24), "flops": 8.0 * rows * v}


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions
def _exact_quantized(y, codes):
    """y in 8 bits as values, from the definition: multiples of a step under each block's largest value."""
    rows, cols = y.shape
    top = F.pad(y.abs(), (0, -cols % 128)).view(rows, -1, 128).amax(2)
    unit = torch.where(top > 0, top / _LARGEST[codes], 1.0).repeat_interleave(128, 1)[:, :cols]
    v = y / unit
    if codes == "int8":
        return torch.round(v) * unit
    # three bits behind the leading one, multiples of 2^-9 at the least
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -40))), min=-6.0) - 3)
    return torch.round(v / step) * step * unit


def _exact_norm(s):
    if s["kind"] == "norm":
        h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        stored = h.to(s["x"].dtype if s["residual"] is None else s["residual"].dtype).double()       # (the norm is that of what is stored)
        rstd = 1 / ((stored * stored).sum(1) / h.shape[1] + EPS).sqrt()
        y = stored * s["w"].double() * rstd[:, None]
        out = dict(rstd=rstd, h=h) if s["residual"] is not None else dict(rstd=rstd)
        if s["y"]:
            out["y"] = y
        if s["codes"] != "none":
            out["quantized"] = _exact_quantized(y, s["codes"])
        return out
    r, n = s["rstd"].double()[:, None], s["h"].shape[1]
    g, h = s["dy"].double() * s["w"].double(), s["h"].double()
    dx = r * g - r * r * r * h * ((g * h).sum(1, keepdim=True) / n)
    return dict(dx=dx if s["dh"] is None else dx + s["dh"].double(), dw=(s["dy"].double() * h * r).sum(0))


def _exact_adapters(s):
    ids, x, s1 = s["ids"].long(), s["x"].double(), s["scaling"].double()
    forward = s["kind"] == "adapters"
    out = s["y"].double() if forward else s["dx"].double()
    dA, dB = torch.zeros(s["A"].shape, dtype=torch.float64, device=x.device), torch.zeros(s["B"].shape, dtype=torch.float64, device=x.device)
    for i in range(s["adapters"]):
        rows = torch.nonzero(ids == i)[:, 0]
        if not len(rows):
            continue
        A, B = s["A"][i].double(), s["B"][i].double()
        if forward:
            out[rows] += s1[i] * torch.mm(torch.mm(x[rows], A.t().contiguous()), B)
            continue
        dy = s["dy"][rows].double()
        v = s1[i] * torch.mm(dy, B.t().contiguous())
        out[rows] += torch.mm(v, A)
        dA[i] = torch.mm(v.t().contiguous(), x[rows])
        dB[i] = s1[i] * torch.mm(s["u"][rows].double().t().contiguous(), dy)
    return out if forward else dict(dx=out, dA=dA, dB=dB)


def _exact_logits(s):
    tokens, parts = s["tokens"], []
    forward = s["kind"] == "log_probabilities"
    for at in range(0, s["rows"], 256):                            # (rows by rows: 64 bits of all of them at once take much memory)
        x, t = s["logits"][at:at + 256].double(), tokens[at:at + 256]
        lse = torch.logsumexp(x, 1) if forward else s["lse"][at:at + 256].double()
        empty = (x == float("-inf")).all(1)
        lp = torch.where(empty[:, None], float("-inf"), x - torch.where(empty, 0.0, lse)[:, None])
        p = torch.exp(lp)
        finite = torch.where(p > 0, lp, 0.0)
        picked = torch.where(t < 0, 0.0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0])
        if forward:
            part = dict(logp=picked, entropy=-(p * finite).sum(1), lse=torch.where(empty, float("-inf"), lse))
            if s["top"]:
                part["indices"] = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
                part["values"] = lp.gather(1, part["indices"])
            parts.append(part)
            continue
        a = torch.where((t < 0) | empty, 0.0, s["dlogp"][at:at + 256].double())
        h, b = s["entropy"][at:at + 256].double(), s["dentropy"][at:at + 256].double()
        dx = F.one_hot(t.clamp(min=0), x.shape[1]) * a[:, None] - p * (a[:, None] + torch.where(p > 0, finite + h[:, None], 0.0) * b[:, None])
        parts.append(dict(dx=dx))
    whole = {k: torch.cat([part[k] for part in parts]) for k in parts[0]}
    return whole if forward else whole["dx"]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    return _exact_norm(s) if kind.startswith("norm") else _exact_adapters(s) if kind.startswith("adapters") else _exact_logits(s)
