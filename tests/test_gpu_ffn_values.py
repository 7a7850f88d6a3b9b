"""The feed-forward operators' values where a looser bound would hide a fault:
exact or relative comparisons, on inputs chosen so that the result is known."""
from __future__ import annotations

import math

import pytest
import torch

from brovisionml_amd import ffn

pytestmark = pytest.mark.gpu
BF, HF, FP, E4 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def say(msg: str) -> None:
    print("[gpu] " + msg, flush=True)


# ---------------------------------------------------------------------------
# the norm's 8-bit output is the quotient, rounded to nearest
# ---------------------------------------------------------------------------
def _integers_of_known_norm(top: int, cols: int):
    """Integers of magnitude <= top, top among them, whose squares sum to
    cols 4^k, so that every sum of squares is exact and rstd is 2^-k; (row, k)."""
    k = max(0, int(math.log2(top)) - 2)
    left, row = cols * 4 ** k - top * top, [top]
    # ratios to top whose quotients by the scale fall on ties of 3 mantissa bits
    for j in (1, 2, 3, 5, 7, 11, 13, 15, 17, 25, 29):
        v = top * j // 32 if top * j % 32 == 0 else top * j // 28
        for x in (v, -(top * j // 4)):
            if 0 < abs(x) <= top and x * x <= left:
                row.append(x)
                left -= x * x
    while left > 0:
        v = min(top, math.isqrt(left))
        row.append(v)
        left -= v * v
    assert left == 0 and len(row) <= cols
    return row + [0] * (cols - len(row)), k


def test_e4m3_is_the_rounded_quotient(cuda):
    say("e4m3 quotients")
    made = [_integers_of_known_norm(top, 256) for top in range(4, 449)]
    x = torch.tensor([r for r, _ in made], dtype=FP)
    y = x * torch.tensor([2.0 ** -k for _, k in made])[:, None]
    scale = y.abs().amax(-1) / 448
    want = (y / scale[:, None]).to(E4)
    got = ffn.add_rms_norm(x.to(cuda), eps=0.0, dtype=E4)
    assert torch.equal(got.scale.cpu(), scale)
    off = got.y.cpu().view(torch.uint8) != want.view(torch.uint8)
    assert not off.any(), f"{int(off.sum())} of {off.numel()} values a step apart"


def test_e4m3_of_a_row_beyond_float32(cuda):
    """A product that overflows leaves an infinite scale, whose quotients are 0
    (the infinite value's: none); what one row holds stays in it."""
    say("e4m3 overflow")
    x = torch.ones(3, 64, device=cuda)
    w = torch.ones(64, device=cuda)
    x[1, 3], w[3] = 60.0, 3e38  # 60 rstd = 7.9: y = 2.4e39
    got = ffn.add_rms_norm(x, None, w, 0.0, dtype=E4)
    assert got.scale[1].isinf() and got.scale[[0, 2]].isfinite().all()
    assert got.y[1, 3].float().isnan()
    others = torch.arange(64, device=cuda) != 3
    assert not got.y[1].float()[others].any() and got.y[[0, 2]].float().isfinite().all()
    assert (got.y[[0, 2], 3].float() == 448).all()
