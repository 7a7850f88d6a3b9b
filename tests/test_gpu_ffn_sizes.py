"""The feed-forward operators at the ends of their sizes: launches of more than
2^32 threads and rows close to the largest 32-bit integer."""
from __future__ import annotations

import pytest
import torch

from brovisionml_amd import _lib, ffn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


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


def _places(n: int, around: int):
    """Indices below n: the first, the last, and those about multiples of
    `around`."""
    some = [torch.arange(min(n, 3000)), torch.arange(max(0, n - 3000), n)]
    some += [torch.arange(k - 300, min(n, k + 300)) for k in range(around, n, around)]
    return torch.cat(some).unique().cuda()


# teams of one wave and of two, more rows than 2^32 threads have at once
@pytest.mark.parametrize("rows,cols", [(2 ** 26 + 9, 8), (2 ** 25 + 3, 513)])
def test_norm_of_more_rows_than_threads_along_a_grid(cuda, rows, cols):
    say(f"norm {rows}x{cols}")
    x = torch.empty(rows, cols, dtype=BF, device=cuda)
    for part in x.split(2 ** 22):
        part.normal_()
    got = ffn.add_rms_norm(x, eps=1e-6, save=True)
    at = _places(rows, 2 ** 22)
    s = x[at].double()
    want = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + 1e-6)
    off = (got.y[at].double() - want).abs()
    assert (off <= want.abs() * (2.0 ** -8 + (cols + 16) * 2.0 ** -23)).all()
    # every row was normed: its squares' mean is 1 but for y's rounding
    for part in got.y.split(2 ** 22):
        mean = part.float().square().mean(-1)
        assert ((mean - 1).abs() <= 2.0 ** -6).all()


def test_both_gradients_of_more_tiles_than_a_launch_holds(cuda):
    """2^30 + 77 rows are 2^24 + 2 tiles of the two gradients' common launch: each
    then goes by itself.  Whole numbers, so that every sum is exact."""
    rows, n, k = 2 ** 30 + 77, 8, 8
    say(f"gradients of {rows} rows")
    tile, deep, _, _ = _lib.ffn_plan(rows, n, k, _lib.BF16, 3)
    assert (tile, deep) == (64, True) and (rows + 63) // 64 >= 2 ** 24
    w = torch.randint(-4, 5, (n, k), device=cuda).to(BF)
    x, dy = (torch.empty(rows, m, dtype=BF, device=cuda) for m in (k, n))
    for part in (*x.split(2 ** 26), *dy.split(2 ** 26)):
        part.random_(-1, 2)
    dx, dw, db = ffn.linear_backward(dy, x, w)
    want_w, want_b = 0, 0
    for i in range(0, rows, 2 ** 25):
        d, part = dy[i:i + 2 ** 25], slice(i, i + 2 ** 25)
        # at most 8 products of up to 4, and 2^25 of up to 1: exact in fp32
        assert torch.equal(dx[part].float(), d.float() @ w.float())
        want_w = want_w + (d.float().t().contiguous() @ x[part].float()).double()
        want_b = want_b + d.sum(0, dtype=torch.float32).double()
    assert float(want_w.abs().max()) < 2 ** 23 and float(want_b.abs().max()) < 2 ** 23
    assert torch.equal(dw, want_w.to(BF)) and torch.equal(db, want_b.to(BF))


def test_no_rows_in_an_inner_dimension(cuda):
    say("no rows")
    x, w = torch.zeros(3, 0, 64, dtype=BF, device=cuda), torch.ones(40, 64, dtype=BF, device=cuda)
    assert ffn.add_rms_norm(x, x).y.shape == x.shape
    y = ffn.linear(x, w, save=True)
    assert y.y.shape == y.z.shape == (3, 0, 40)
    assert ffn.gated(x, w).y.shape == (3, 0, 20)
    dx, dw, db = ffn.linear_backward(y.y, x, w)
    assert dx.shape == x.shape and not dw.any() and not db.any()
