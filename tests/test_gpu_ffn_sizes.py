"""The feed-forward operators at the ends of their sizes: launches of more than
2^32 threads and rows close to the largest 32-bit integer."""
from __future__ import annotations

import pytest
import torch

from brovisionml_amd import ffn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def say(msg: str) -> None:
    print("[gpu] " + msg, flush=True)


def test_bias_gradient_of_the_most_rows(cuda):
    """Ones in the first and in the last rows of 2^31 - 512: the last run of rows
    ends beyond what an int holds."""
    rows = 2 ** 31 - 512
    say(f"bias gradient of {rows} rows")
    z = torch.zeros(rows, 1, dtype=BF, device=cuda)
    dy = torch.zeros(rows, 1, dtype=BF, device=cuda)
    dy[:40], dy[-88:] = 1, 1
    db = ffn.linear_backward(dy, z, torch.zeros(1, 1, dtype=BF, device=cuda), z, "silu",
                             need_x=False, need_w=False)[2]
    assert float(db) == 64.0  # silu'(0) = 1/2
