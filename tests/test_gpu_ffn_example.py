"""examples/feed_forward.py: the three operators as a program uses them, against
the block's formula in double precision."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from tests import ffn_oracle as orc

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "feed_forward.py")


def load():
    spec = importlib.util.spec_from_file_location("feed_forward", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def formula(block, x, residual):
    s = x.double() + residual.double()
    y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + block.eps) * block.norm_weight.double()
    g, u = (y @ block.w_in.double().t().contiguous() + block.b_in.double()).chunk(2, -1)
    h = orc.act(block.act, g) * u
    return s, h @ block.w_out.double().t().contiguous() + block.b_out.double()


@pytest.mark.parametrize("tokens", [1, 4, 100, 247])
def test_example(cuda, tokens):
    m = load()
    block = m.random_block(256, 680)
    x, r, t = (torch.randn(tokens, 256, device="cuda").bfloat16() for _ in range(3))
    s, part = formula(block, x, r)
    out = block.forward(x, r)
    # norm, products, gate and sum each round once to 8 bits: a few 2^-8 of the
    # part they make, and one 2^-8 of the whole
    scale = part.abs().max() * 4 * 2.0 ** -8
    assert (out.double() - (s + part)).abs().max() <= scale + (s + part).abs().max() * 2.0 ** -8
    w, ws = m.quantised(block.w_in)
    eight = m.forward_8_bits(block, w, ws, x, r)
    # two e4m3 operands: 2^-4 of a value at most each, in sums of 256 of random
    # sign; 10% of the part's size is three times what that leaves
    off = (eight.double() - (s + part)).norm() / part.norm()
    assert off <= 0.1, float(off)
    loss, dx = m.train_step(block, x, r, t)
    want = float(((out.double() - t.double()) ** 2).sum() / (2 * tokens))
    assert abs(loss - want) <= 1e-5 * want and dx.shape == x.shape and dx.isfinite().all()
    # a small step against the gradient: downhill
    assert m.train_step(block, x, r, t)[0] < loss
