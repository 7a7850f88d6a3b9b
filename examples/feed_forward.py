"""The feed-forward half of a pre-norm transformer block over the patches of a
60x80 grid: one training step, then single tokens, then the same in 8 bits.

  python examples/feed_forward.py [--grid H W] [--width K] [--hidden N]

Needs the native library (python -m brovisionml_amd.build) and an MI355X.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from brovisionml_amd import ffn  # noqa: E402


def random_block(width: int, hidden: int, seed: int = 0) -> ffn.FeedForward:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape, std):
        return (torch.randn(shape, generator=g, device="cuda") * std).bfloat16()

    return ffn.FeedForward(1 + randn(width, std=0.1), randn(2 * hidden, width, std=width ** -0.5),
                           randn(width, hidden, std=hidden ** -0.5),
                           randn(2 * hidden, std=0.1), randn(width, std=0.1))


def train_step(block: ffn.FeedForward, x, residual, target, rate: float = 1e-3):
    """One step of plain gradient descent on half the square error a token;
    returns that and the gradient that goes on to the layer before."""
    out, saved = block.forward(x, residual, save=True)
    off = out.float() - target.float()
    grads = block.backward((off / len(off)).to(out.dtype), saved)
    for name, grad in grads.items():
        if name != "x":
            getattr(block, name).sub_(grad, alpha=rate)
    return float((off * off).sum() / (2 * len(off))), grads["x"]


def quantised(w):
    """A weight as e4m3 with a scale a row."""
    scale = (w.float().abs().amax(-1) / 448.0).clamp(min=2.0 ** -126)
    return (w.float() / scale[:, None]).to(torch.float8_e4m3fn), scale


def forward_8_bits(block: ffn.FeedForward, w_in, w_scale, x, residual):
    """The block with its first product in 8 bits: the norm leaves its rows as
    e4m3 with their scales, as the product reads them."""
    n = ffn.add_rms_norm(x, residual, block.norm_weight, block.eps, dtype=torch.float8_e4m3fn)
    h = ffn.gated(n.y, w_in, block.b_in, block.act, x_scale=n.scale, w_scale=w_scale,
                  dtype=x.dtype)
    return ffn.linear(h.y, block.w_out, block.b_out, residual=n.stream).y


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--grid", type=int, nargs=2, default=(60, 80))
    p.add_argument("--width", type=int, default=1280)
    p.add_argument("--hidden", type=int, default=5120)
    a = p.parse_args()
    tokens = a.grid[0] * a.grid[1]
    block = random_block(a.width, a.hidden)
    x, residual, target = (torch.randn(tokens, a.width, device="cuda").bfloat16()
                           for _ in range(3))
    for step in range(3):
        loss, _ = train_step(block, x, residual, target)
        print(f"training step {step}: half the square error a token {loss:.2f}")
    whole = block.forward(x, residual)
    one = block.forward(x[:1].contiguous(), residual[:1].contiguous())
    print(f"a single token against the batch: {float((one - whole[:1]).abs().max()):.4f} off")
    w_in, w_scale = quantised(block.w_in)
    eight = forward_8_bits(block, w_in, w_scale, x, residual)
    off = (eight.float() - whole.float()).norm() / (whole.float() - x.float()
                                                    - residual.float()).norm()
    print(f"8-bit first product: {100 * float(off):.1f}% of the block's contribution off")


if __name__ == "__main__":
    main()
