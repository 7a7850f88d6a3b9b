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


# ---------------------------------------------------------------------------
# activations: relative to their own value
# ---------------------------------------------------------------------------
ULP = 2.0 ** -24  # half a unit in the last place of fp32, relative


def _reference(name, z):
    """(act, its derivative) in double; each tail by itself, where it does not
    cancel."""
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a = 2 * math.sqrt(2 / math.pi)
        p = torch.sigmoid(a * (z + 0.044715 * z ** 3))
        return z * p, p + z * p * (1 - p) * a * (1 + 3 * 0.044715 * z * z)
    p = torch.sigmoid(z)
    return z * p, p + z * p * (1 - p)


def _relative(name, z):
    """How far fp32 may be from act(z), relative to it, and the smallest value
    that an fp32 tail can hold.

    The tail is 2^t, and t's own roundings (its constants, products and
    additions, five at most) are each |t| ln 2 ULP of it; then come an
    exponential and a reciprocal of 2 ULP each (one unit), GELU's polynomial
    (eight fused steps whose terms add up to less than twice its value: 16 ULP,
    and 2 ULP of fit) and three products.  Below 2^-126 a factor of x may be
    zero: |x| 2^-126, with |x| < 128."""
    t = {"gelu": z * z / 2, "gelu_tanh": 1.6 * (z.abs() + 0.045 * z.abs() ** 3),
         "silu": z.abs()}[name]
    return (5 * t + 28) * ULP, 2.0 ** -119


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
def test_activation_tails_keep_their_relative_accuracy(cuda, name):
    say(f"tails of {name}")
    far = 90 if name == "silu" else 14
    z = torch.cat([torch.linspace(-far, 14, 9001, device="cuda"),
                   -torch.logspace(-6, 1, 301, device="cuda")]).to(BF)
    got = ffn.linear(z[:, None], torch.ones(1, 1, device="cuda", dtype=BF), act=name,
                     dtype=FP).y[:, 0].double()
    z = z.double()
    want, _ = _reference(name, z)
    rel, floor = _relative(name, z)
    bad = ~((got - want).abs() <= rel * want.abs() + floor)
    worst = ((got - want).abs() / want.abs().clamp(min=floor)).max()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, {float(worst):.3g} relative"


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
def test_gated_gradient_keeps_the_tails(cuda, name):
    """db of one row is [dh u act'(g), dh act(g)], rounded once to float16."""
    say(f"gated gradient, tails of {name}")
    g = torch.linspace(-6, 6, 4001, device="cuda").to(HF)[None]
    n = g.shape[1]
    x, w = torch.zeros(1, 8, device="cuda", dtype=HF), torch.zeros(2 * n, 8, device="cuda", dtype=HF)
    dh = torch.full((1, n), 512.0, device="cuda", dtype=HF)
    _, _, db = ffn.gated_backward(dh, x, w, torch.cat([g, torch.ones_like(g)], 1), name,
                                  need_x=False, need_w=False)
    value, slope = _reference(name, g[0].double())
    rel, floor = _relative(name, g[0].double())
    # the slope's two terms cancel near its root: relative to their sizes
    size = slope.abs() + 2 * value.abs() * (1 + g[0].double().abs())
    for got, want, off in ((db[:n], 512 * slope, 512 * rel * size),
                           (db[n:], 512 * value, 512 * rel * value.abs())):
        bound = off + 2.0 ** -11 * (want.abs() + off) + 2.0 ** -25 + 512 * floor
        bad = ~((got.double() - want).abs() <= bound)
        assert not bad.any(), int(bad.sum())


@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_of_the_largest_arguments(cuda, name):
    """act' is 1 above and 0 below (none: 1) however large z is."""
    say(f"largest arguments of {name}")
    z = torch.tensor([s * 2.0 ** k for s in (1, -1) for k in range(6, 128)], device="cuda").to(BF)
    n = len(z)
    x, w = torch.zeros(1, 8, device="cuda", dtype=BF), torch.zeros(n, 8, device="cuda", dtype=BF)
    dy = torch.ones(1, n, device="cuda", dtype=BF)
    db = ffn.linear_backward(dy, x, w, z[None], name, need_x=False, need_w=False)[2].float()
    want = torch.ones_like(db) if name == "none" else (z > 0).float()
    # (2^6 is so far out that the tails are below 2^-60)
    assert (db - want).abs().max() <= 2.0 ** -60
    db = ffn.gated_backward(dy, x, torch.cat([w, w]), torch.cat([z, torch.ones_like(z)])[None],
                            name, need_x=False, need_w=False)[2].float()
    assert (db[:n] - want).abs().max() <= 2.0 ** -60
    assert torch.equal(db[n:][want > 0], z.float()[want > 0])
    assert not (db[n:][want == 0].abs() > 2.0 ** -60).any() and not db[n:].isnan().any()


# ---------------------------------------------------------------------------
# products of the smallest numbers, and of no numbers
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("M", [1, 2, 3, 4, 7, 20, 40, 130, 300])
def test_float16_subnormals_are_numbers(cuda, M):
    """Integers times 2^-24 by small powers of two: every sum is exact."""
    say(f"subnormals, {M} rows")
    g = torch.Generator(device="cuda").manual_seed(M)
    tiny = torch.randint(-1023, 1024, (48, 72), generator=g, device="cuda")
    two = 2.0 ** torch.randint(0, 3, (M, 72), generator=g, device="cuda")
    w, x = (tiny * 2.0 ** -24).to(HF), two.to(HF)
    assert torch.equal(w.double(), tiny * 2.0 ** -24)
    want = two.double() @ (tiny.double().t().contiguous() * 2.0 ** -24)
    assert torch.equal(ffn.linear(x, w, dtype=FP).y.double(), want)
    both = ffn.gated(x, torch.cat([w, torch.ones_like(w)]), act="none", dtype=FP).y.double()
    assert torch.equal(both, want * two.double().sum(-1, keepdim=True))
    # subnormal dz by rows of W and of x, results rounded once to float16
    dz = (torch.randint(-1023, 1024, (M, 48), generator=g, device="cuda") * 2.0 ** -24).to(HF)
    four = (2.0 ** torch.randint(0, 3, (48, 72), generator=g, device="cuda")).to(HF)
    dx, dw, db = ffn.linear_backward(dz, x, four)
    assert torch.equal(dx, (dz.double() @ four.double()).to(HF))
    assert torch.equal(dw, (dz.double().t().contiguous() @ x.double()).to(HF))
    assert torch.equal(db, dz.double().sum(0).to(HF))


@pytest.mark.parametrize("dtype", [BF, HF, E4], ids=["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 17, 33, 150])
def test_no_numbers_stay_in_their_rows(cuda, M, dtype):
    say(f"NaN, {M} rows, {dtype}")
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, 144, generator=g, device="cuda")
    w = torch.randn(50, 144, generator=g, device="cuda")
    x[M // 2, 131] = float("nan")
    w[7, 5] = float("nan")
    kw = {}
    if dtype == E4:
        kw = dict(x_scale=torch.ones(M, device="cuda"), w_scale=torch.ones(50, device="cuda"),
                  dtype=FP)
    y = ffn.linear(x.to(dtype), w.to(dtype), **kw).y
    want = torch.zeros(M, 50, dtype=torch.bool, device="cuda")
    want[M // 2] = True
    want[:, 7] = True
    assert torch.equal(y.isnan(), want)
