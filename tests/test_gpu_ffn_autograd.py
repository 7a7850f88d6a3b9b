"""The feed-forward operators recorded by autograd: the gradients of their own
backward functions, bit for bit, and refusals where there are none."""
from __future__ import annotations

import pytest
import torch

from brovisionml_amd import ffn

pytestmark = pytest.mark.gpu
BF, HF, FP, E4 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def say(msg: str) -> None:
    print("[gpu] " + msg, flush=True)


def leaves(*shapes, dtype=BF, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=g, device="cuda").div(4).to(dtype).requires_grad_()
            for s in shapes]


@pytest.mark.parametrize("save", [False, True])
@pytest.mark.parametrize("name,rows,bias_type,out", [
    ("none", 1, BF, BF), ("gelu", 3, FP, FP), ("silu", 40, BF, BF), ("relu", 200, FP, BF)])
def test_linear_is_recorded(cuda, name, rows, bias_type, out, save):
    say(f"linear {name} {rows}")
    x, w, r = leaves((rows, 72), (40, 72), (rows, 40))
    b, = leaves((40,), dtype=bias_type, seed=1)
    res = r.to(out)
    y, z = ffn.linear(x, w, b, name, res, dtype=out, save=save)
    assert y.requires_grad and (z is not None) == save and (z is None or not z.requires_grad)
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, (x, w, b, r), dy)
    with torch.no_grad():
        plain = ffn.linear(x, w, b, name, res, dtype=out, save=True)
        assert torch.equal(plain.y, y) and not plain.y.requires_grad
        dx, dw, db = ffn.linear_backward(dy, x, w, None if name == "none" else plain.z, name)
    for a, want in zip(got, (dx, dw, db.to(bias_type), dy.to(BF))):
        assert a.dtype == want.dtype and torch.equal(a, want)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("shape", [(2, 72), (3, 20, 72)])
def test_gated_is_recorded(cuda, shape, dtype):
    say(f"gated {shape} {dtype}")
    x, w, b = leaves(shape, (80, 72), (1, 80), dtype=dtype)
    h = ffn.gated(x, w, b, "gelu_tanh").y
    got = torch.autograd.grad(h.sum(), (x, w, b))  # (an expanded gradient of ones)
    with torch.no_grad():
        plain = ffn.gated(x, w, b, "gelu_tanh", save=True)
        want = ffn.gated_backward(torch.ones_like(h), x, w, plain.z, "gelu_tanh")
    assert torch.equal(h, plain.y)
    for a, v in zip(got, want):
        assert torch.equal(a.reshape(v.shape), v)
    assert got[2].shape == (1, 80)


@pytest.mark.parametrize("xt,yt", [(BF, BF), (FP, FP), (FP, HF)])
def test_norm_is_recorded(cuda, xt, yt):
    say(f"norm {xt} to {yt}")
    x, r, w = leaves((33, 264), (33, 264), (264,), dtype=xt)
    n = ffn.add_rms_norm(x, r, w, dtype=yt)
    dy, ds = torch.randn_like(n.y), torch.randn_like(n.stream)
    with torch.no_grad():
        p = ffn.add_rms_norm(x, r, w, dtype=yt, save=True)
        assert torch.equal(p.y, n.y) and torch.equal(p.stream, n.stream)
        both = ffn.add_rms_norm_backward(dy, p.stream, w, p.rstd, ds)
        only = ffn.add_rms_norm_backward(dy, p.stream, w, p.rstd)
    got = torch.autograd.grad((n.y, n.stream), (x, r, w), (dy, ds), retain_graph=True)
    assert torch.equal(got[0], both[0]) and torch.equal(got[1], both[0])
    assert torch.equal(got[2], both[1])
    got = torch.autograd.grad(n.y, (x, w), dy, retain_graph=True)
    assert torch.equal(got[0], only[0]) and torch.equal(got[1], only[1])
    got = torch.autograd.grad(n.stream, (x, w), ds)  # the norm itself unused
    assert torch.equal(got[0], ds) and not got[1].any()
    # without a residual the stream is x itself
    n = ffn.add_rms_norm(x, None, w, dtype=yt, save=True)
    assert n.stream is x and n.rstd is not None and not n.rstd.requires_grad
    with torch.no_grad():
        want = ffn.add_rms_norm_backward(dy, x, w, n.rstd)
    got = torch.autograd.grad(n.y, (x, w), dy)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_block_is_recorded(cuda):
    """A block of parameters under autograd against its own backward()."""
    say("block")
    wn, wi, wo, bi, bo = leaves((72,), (96, 72), (72, 48), (96,), (72,))
    x, r = leaves((50, 72), (50, 72), seed=2)
    block = ffn.FeedForward(wn, wi, wo, bi, bo)
    out = block.forward(x, r)
    dout = torch.randn_like(out)
    out.backward(dout)
    with torch.no_grad():
        again, saved = block.forward(x, r, save=True)
        g = block.backward(dout, saved)
    assert torch.equal(out, again)
    for t, name in ((wn, "norm_weight"), (wi, "w_in"), (wo, "w_out"), (bi, "b_in"), (bo, "b_out"),
                    (x, "x"), (r, "x")):
        assert torch.equal(t.grad, g[name]), name


def test_what_has_no_gradient_is_refused(cuda):
    say("refusals")
    x, w, r = leaves((5, 64), (40, 64), (5, 40))
    with pytest.raises(RuntimeError, match="ffn ops: add_rms_norm: float8 output has no gradient"):
        ffn.add_rms_norm(x, dtype=E4)
    with pytest.raises(RuntimeError, match="ffn ops: linear: a given output has no gradient"):
        ffn.linear(x, w, out=torch.empty_like(r))
    one = torch.ones(40, device="cuda")
    with pytest.raises(RuntimeError, match="ffn ops: gated: float8 operands have no gradient"):
        ffn.gated(x.detach().to(E4), w.detach().to(E4), one.clone().requires_grad_(),
                  x_scale=one[:5], w_scale=one)
    y = ffn.linear(x, w, act="silu").y
    dx, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()
    with torch.no_grad():  # as before
        assert ffn.add_rms_norm(x, dtype=E4).y.dtype == E4
        assert not ffn.linear(x, w, out=torch.empty_like(r)).y.requires_grad
    assert not ffn.linear(x.detach(), w.detach()).y.requires_grad
