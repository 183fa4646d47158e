"""A feed-forward block x + W2 gelu(W1 norm(x) + c1) + c2, trained with its activations kept in 8 bits.

Of the forward pass stay, for a token: xhat (for the norm's gradient and for W1's), the argument of gelu, and its value (for W2's), each at
1.03 bytes an element, and rstd.  The products are bf16 with fp32 accumulators, the parameters and their gradients fp32.

    python examples/feed_forward_training.py [--tokens 8192 --width 2048 --hidden 8192 --steps 20 --rate 2e-4 --keep int8]
"""
import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import qgemm_amd as Q  # noqa: E402


def _product(a, W, layout, n, dtype=torch.bfloat16):
    return Q.gemm(a, W, torch.empty(a.shape[0], n, dtype=dtype, device=a.device), layout)


class NormLinear(torch.autograd.Function):
    """norm(x) W^T + c for x [tokens, width] bf16: one checkpoint of xhat serves the weight's gradient and the norm's."""

    @staticmethod
    def forward(ctx, x, w, b, W, c, keep):
        y, _, rstd, q, scales = Q.layer_norm(x, w, b, keep=keep)
        half = W.bfloat16()
        ctx.save_for_backward(q, scales, rstd, w, b, half)
        return _product(y, half, "nk", W.shape[0]).add_(c)

    @staticmethod
    def backward(ctx, dz):
        q, scales, rstd, w, b, half = ctx.saved_tensors
        dz = dz.contiguous()
        dW, dc = Q.weight_gradient(dz, q, scales, w, b)
        dy = _product(dz, half, "kn", half.shape[1], torch.float32)
        dx, dw, db = Q.layer_norm_backward(dy, q, None, rstd, w, scales=scales, out_dtype=dz.dtype)
        return dx, dw, db, dW, dc, None


class Gelu(torch.autograd.Function):
    """gelu(z), of which z is kept in 8 bits."""

    @staticmethod
    def forward(ctx, z, keep):
        ctx.save_for_backward(*Q.checkpoint(z, keep))
        return F.gelu(z)

    @staticmethod
    def backward(ctx, dh):
        z = Q.restore(*ctx.saved_tensors, torch.float32)
        inside = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return (dh * (inside + z * torch.exp(-0.5 * z * z) * (0.5 / torch.pi) ** 0.5)).to(dh.dtype), None


class Linear(torch.autograd.Function):
    """h W^T + c, of which h is kept in 8 bits."""

    @staticmethod
    def forward(ctx, h, W, c, keep):
        half = W.bfloat16()
        ctx.save_for_backward(*Q.checkpoint(h, keep), half)
        return _product(h, half, "nk", W.shape[0]).add_(c)

    @staticmethod
    def backward(ctx, dz):
        q, scales, half = ctx.saved_tensors
        dz = dz.contiguous()
        dW, dc = Q.weight_gradient(dz, q, scales)
        return _product(dz, half, "kn", half.shape[1]), dW, dc, None


class FeedForward(torch.nn.Module):
    def __init__(self, width, hidden, keep=torch.int8, device="cuda"):
        super().__init__()
        self.keep = keep
        self.norm = torch.nn.LayerNorm(width, device=device)
        self.up, self.down = torch.nn.Linear(width, hidden, device=device), torch.nn.Linear(hidden, width, device=device)

    def forward(self, x):
        z = NormLinear.apply(x, self.norm.weight, self.norm.bias, self.up.weight, self.up.bias, self.keep)
        return x + Linear.apply(Gelu.apply(z, self.keep), self.down.weight, self.down.bias, self.keep)


def train(tokens, width, hidden, steps, keep, rate=1e-3, seed=0):
    """Losses of `steps` steps towards what another block of the same sizes gives."""
    torch.manual_seed(seed)
    block, aim = FeedForward(width, hidden, keep), FeedForward(width, hidden, keep)
    optimizer = torch.optim.AdamW(block.parameters(), lr=rate)
    losses = []
    for _ in range(steps):
        x = torch.randn(tokens, width, device="cuda", dtype=torch.bfloat16)
        with torch.no_grad():
            target = aim(x)
        loss = (block(x) - target).float().square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("tokens", 8192), ("width", 2048), ("hidden", 8192), ("steps", 20)):
        parser.add_argument("--" + name, type=int, default=value)
    parser.add_argument("--rate", type=float, default=2e-4)
    parser.add_argument("--keep", choices=("int8", "float8_e4m3fn"), default="int8")
    args = parser.parse_args()
    losses = train(args.tokens, args.width, args.hidden, args.steps, getattr(torch, args.keep), args.rate)
    kept = args.width + 2 * args.hidden
    print(f"kept of a token: {kept + 4 * (-(-args.width // 128) + 2 * -(-args.hidden // 128)) + 4} bytes, in bf16 {2 * kept}")
    print("loss:", " ".join(f"{loss:.5f}" for loss in losses))


if __name__ == "__main__":
    main()
