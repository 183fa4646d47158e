"""The operators beside the products together, as a model uses them: a decoding step on 8-bit weights with adapters, and a policy's update of adapters and norms."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import qgemm_amd as Q
from qgemm_amd.lib import check, load_library
from tests import training_ref as R
from tests.util import say

pytestmark = pytest.mark.gpu

F32, BF16, I8, F8 = torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def randn(*shape, seed, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_a_decoding_step_on_8_bit_weights(rows, codes):
    """residual + rms_norm -> codes -> block-scaled product, adapters beside it -> rms_norm -> logits -> log probabilities, against 64 bits out of the same codes: what is
    left are 16-bit roundings of y, z (2^-9 on average 0.3 of it) and sums, together below 0.01 of the logits' spread."""
    say("chain decoding", rows, codes)
    k, n, vocabulary, adapters, rank = 512, 384, 3000, 6, 16
    x, residual, w1, w2 = randn(rows, k, seed=1), randn(rows, k, seed=2), 1 + randn(k, seed=3, scale=0.1, dtype=F32), 1 + randn(n, seed=4, scale=0.1, dtype=F32)
    A, B, s = randn(adapters, rank, k, seed=5, scale=k ** -0.5), randn(adapters, rank, n, seed=6, scale=0.2), torch.linspace(0.5, 1.5, adapters, device="cuda")
    W, head = randn(n, k, seed=7, scale=k ** -0.5), randn(vocabulary, n, seed=8, scale=2 * n ** -0.5)
    ids = torch.randint(-1, adapters, (rows,), generator=torch.Generator().manual_seed(9)).cuda()
    wq, ws = Q.quantize(W, codes, Q.QUANT_BLOCK_128x128)

    def step():
        groups = Q.group_rows(ids, adapters)
        y, h, _, q, scales = Q.rms_norm(x, w1, residual=residual, codes=codes)
        z = torch.empty(rows, n, dtype=BF16, device="cuda")
        Q.scaled_gemm(q, wq, scales, ws, z, rows, n, k, Q.SCALE_BLOCK128)
        Q.add_adapters(z, y, A, B, groups, s, out=z)
        t = Q.rms_norm(z, w2)[0]
        logits = Q.gemm(t, head, torch.empty(rows, vocabulary, dtype=F32, device="cuda"), "nk")
        return y, h, q, scales, z, logits, Q.log_probabilities(logits, logits.argmax(-1), top=4)

    y, h, q, scales, z, logits, (logp, entropy, lse, values, indices) = step()
    d = lambda t: t.double().cpu()  # noqa: E731
    assert torch.equal(h, (x.float() + residual.float()).bfloat16())
    real = d(wq.float()) * d(ws).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    Z = torch.from_numpy(R.values(q, scales)) @ real.t()
    for t, i in enumerate(ids.tolist()):
        if i >= 0:
            Z[t] += d(s)[i] * (d(y)[t] @ d(A)[i].t()) @ d(B)[i]
    T = Z / (Z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * d(w2)
    want = T @ d(head).t()
    assert ((d(logits) - want).square().mean().sqrt() / want.std()).item() <= 0.01
    L = torch.log_softmax(d(logits), -1)
    top = torch.sort(d(logits), dim=-1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(indices.cpu(), top) and torch.equal(values[:, 0], logp)
    assert torch.allclose(d(values), L.gather(-1, top), atol=1e-5) and torch.allclose(d(entropy), -(L.exp() * L).sum(-1), atol=1e-5)

    # the same in a graph, with other inputs at every replay
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (11, 12, 13):
        x.copy_(randn(rows, k, seed=seed))
        ids.copy_(torch.randint(-1, adapters, (rows,), generator=torch.Generator().manual_seed(seed)).cuda())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*out[:6], *out[6])]
        again = step()
        assert all(torch.equal(a, b) for a, b in zip(got, (*again[:6], *again[6])))


# Against the root of the mean square: each gradient passes through at most eight bf16 roundings of independent errors (h, y, z, logits' gradient, and those of the gradients on
# their way back), each 2^-9 at most and 0.6 of that on average: 8^0.5 * 0.0012 = 0.0033, and the norm and the softmax pass an error on at most threefold.
@pytest.mark.parametrize("rows, k, n, vocabulary", [(300, 256, 384, 1000), (77, 200, 264, 777), (1, 128, 128, 500)])
def test_gradients_of_a_policys_update(rows, k, n, vocabulary):
    say("chain gradients", rows, k, n, vocabulary)
    adapters, rank = 3, 8
    x, w1, w2 = randn(rows, k, seed=21), 1 + randn(k, seed=22, scale=0.1, dtype=F32), 1 + randn(n, seed=23, scale=0.1, dtype=F32)
    A, B, s = randn(adapters, rank, k, seed=24, scale=k ** -0.5), randn(adapters, rank, n, seed=25, scale=0.3), torch.tensor([0.5, 1.0, 2.0], device="cuda")
    W, head = randn(n, k, seed=26, scale=k ** -0.5), randn(vocabulary, n, seed=27, scale=n ** -0.5)
    ids = torch.randint(-1, adapters, (rows,), generator=torch.Generator().manual_seed(28)).cuda()
    tokens = torch.randint(0, vocabulary, (rows,), generator=torch.Generator().manual_seed(29)).cuda()
    advantage, bonus = randn(rows, seed=30, dtype=F32), torch.full((rows,), 0.01, device="cuda")

    groups = Q.group_rows(ids, adapters)
    y, _, rstd1 = Q.rms_norm(x, w1)
    z, u = Q.add_adapters(Q.gemm(y, W, torch.empty(rows, n, dtype=BF16, device="cuda"), "nk"), y, A, B, groups, s, keep=True)
    t, _, rstd2 = Q.rms_norm(z, w2)
    logits = Q.gemm(t, head, torch.empty(rows, vocabulary, dtype=F32, device="cuda"), "nk")
    logp, entropy, lse = Q.log_probabilities(logits, tokens)
    dlogits = Q.log_probabilities_backward(logits, tokens, lse, entropy, advantage, bonus, BF16)
    dt = Q.gemm(dlogits, head, torch.empty(rows, n, dtype=F32, device="cuda"), "kn")
    dz, dw2 = Q.rms_norm_backward(dt, z, rstd2, w2, out_dtype=BF16)
    dy, dA, dB = Q.add_adapters_backward(dz, y, u, A, B, groups, s, dx=Q.gemm(dz, W, torch.empty(rows, k, dtype=F32, device="cuda"), "kn"))
    dx, dw1 = Q.rms_norm_backward(dy, x, rstd1, w1, dh=x)

    wide = {name: v.double().cpu().requires_grad_() for name, v in dict(x=x, w1=w1, w2=w2, A=A, B=B).items()}
    norm = lambda v, w: v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w  # noqa: E731
    Y = norm(wide["x"], wide["w1"])
    which = F.one_hot(ids.cpu() + 1, adapters + 1)[:, 1:].double()
    delta = torch.einsum("ta,tr,arn->tn", which * s.cpu().double(), torch.einsum("tk,ark,ta->tr", Y, wide["A"], which), wide["B"])
    L = torch.log_softmax(norm(Y @ W.double().cpu().t() + delta, wide["w2"]) @ head.double().cpu().t(), -1)
    picked = L[torch.arange(rows), tokens.cpu()]
    H = -(L.exp() * L).sum(-1)
    ((picked * advantage.cpu()).sum() + (H * bonus.cpu()).sum() + 0.5 * wide["x"].square().sum()).backward()
    assert torch.allclose(logp.double().cpu(), picked, atol=0.05) and torch.allclose(entropy.double().cpu(), H, atol=0.05)
    for name, got in dict(x=dx, w1=dw1, w2=dw2, A=dA, B=dB).items():
        want = wide[name].grad
        error = ((got.double().cpu() - want).norm() / want.norm().clamp(min=1e-30)).item()
        assert error <= 0.02 or want.norm() == 0 == got.norm(), f"{name}: {error}"


@pytest.mark.parametrize("wanted", ["dx", "dA", "dB", "dx dA", "dA dB"])
def test_parts_of_the_backward_pass(wanted):
    """The C entry computes what it is asked for, with the bits of the whole pass."""
    say("add_adapters_backward parts", wanted)
    rows, adapters, rank, k, n = 150, 4, 24, 2048, 1024
    x, dy, A, B = randn(rows, k, seed=31), randn(rows, n, seed=32), randn(adapters, rank, k, seed=33), randn(adapters, rank, n, seed=34)
    u, groups = randn(rows, rank, seed=35, dtype=F32), Q.group_rows(torch.randint(-1, adapters, (rows,), generator=torch.Generator().manual_seed(36)).cuda(), adapters)
    whole = dict(zip(("dx", "dA", "dB"), Q.add_adapters_backward(dy, x, u, A, B, groups)))
    out = {name: torch.full_like(t, 7) for name, t in whole.items()}
    at = lambda name: out[name].data_ptr() if name in wanted.split() else None  # noqa: E731
    check(load_library().qgemm_add_adapters_backward(
        Q.DT_BF16, Q.DT_BF16, Q.DT_F32, dy.data_ptr(), n, x.data_ptr(), k, u.data_ptr() if "dB" in wanted else None, A.data_ptr(), B.data_ptr(), None, groups.words.data_ptr(), None,
        k, at("dx"), k, at("dA"), at("dB"), rows, adapters, rank, k, n, Q.ops._stream()))
    for name, t in out.items():
        assert torch.equal(t, whole[name]) if name in wanted.split() else (t == 7).all(), name


def test_calls_on_several_streams_at_once():
    """More streams than have a workspace block of their own, all at work on calls that need one."""
    say("chain streams")
    rows, adapters, rank, k, n = 400, 5, 16, 1024, 1024
    sets = []
    for i in range(5):
        sets.append((randn(rows, k, seed=40 + i), randn(rows, n, seed=50 + i), randn(adapters, rank, k, seed=60 + i), randn(adapters, rank, n, seed=70 + i),
                     torch.randint(-1, adapters, (rows,), generator=torch.Generator().manual_seed(i)).cuda(), randn(4, 60000, seed=80 + i, dtype=F32)))

    def work(x, y, A, B, ids, logits):
        groups = Q.group_rows(ids, adapters)
        out, u = Q.add_adapters(y, x, A, B, groups, keep=True)
        h, _, rstd = Q.rms_norm(out)
        return (out, u, *Q.add_adapters_backward(h, x, u, A, B, groups), *Q.rms_norm_backward(h, out, rstd, torch.ones(n, device="cuda")),
                *Q.log_probabilities(logits, torch.arange(4, device="cuda"), top=8))

    want = [work(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(work(*s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
        del got
