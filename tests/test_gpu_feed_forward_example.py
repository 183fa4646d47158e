"""The training example: its gradients against 64-bit autograd of the same block, and its loss."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "feed_forward_training.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("feed_forward_training", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


# Against the root of the mean square: xhat, z and h lie in blocks whose largest value is 2.5 - 4 deviations, so that a unit of int8 is at most
# 4 / 63.5 = 0.063 of a deviation and its rounding 0.063 / sqrt(12) = 0.018; e4m3 rounds by at most 2^-4, 0.036 on average.  A gradient takes
# two such roundings (an activation, and the slope of gelu) and bf16 ones of 0.003: together below 0.03 and 0.055.
@pytest.mark.parametrize("keep, bound", [(torch.int8, 0.03), (torch.float8_e4m3fn, 0.055)])
@pytest.mark.parametrize("tokens, width, hidden", [(300, 256, 384), (77, 200, 264), (1, 128, 128)])
def test_gradients_of_the_block(example, tokens, width, hidden, keep, bound):
    torch.manual_seed(tokens)
    block = example.FeedForward(width, hidden, keep)
    x = torch.randn(tokens, width, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(tokens, width, device="cuda", dtype=torch.bfloat16)
    block(x).backward(dy)
    got = {"x": x.grad, **{name: p.grad for name, p in block.named_parameters()}}

    wide = {name: p.detach().double().cpu().requires_grad_() for name, p in block.named_parameters()}
    X = x.detach().double().cpu().requires_grad_()
    y = F.layer_norm(X, (width,), wide["norm.weight"], wide["norm.bias"])
    z = y @ wide["up.weight"].t() + wide["up.bias"]
    (X + F.gelu(z) @ wide["down.weight"].t() + wide["down.bias"]).backward(dy.double().cpu())
    want = {"x": X.grad, **{name: p.grad for name, p in wide.items()}}
    for name, g in want.items():
        error = ((got[name].double().cpu() - g).norm() / g.norm()).item()
        assert error <= bound, f"{name}: {error}"


def test_the_loss_falls(example):
    losses = example.train(512, 256, 512, 30, torch.int8)
    assert losses[-1] < 0.5 * losses[0], losses
