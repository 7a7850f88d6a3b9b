"""The feed-forward operators' definitions in double precision, plain torch, and
the rounding bounds of an fp32 computation that stores 16 bits: the oracle of
tests/test_gpu_ffn.py.

Bounds, per element, derived from the arithmetic and not from results (u = the
stored type's unit roundoff, f = 2^-23, one truncated fp32 addition):
a product of K terms is off by at most (K + 8) f sum |x w|; an activation
follows its argument with a slope of at most 1.13 and is itself off by at most
8 f |z| + 2e-7 |z| (the normal distribution's formula 1.5e-7, exp and
reciprocal an ulp each); its derivative by 2e-6 (1 + |z|); and the store
adds u |value| plus half the smallest subnormal.  The 8-bit matrix
instruction sums eight neighbouring products at a time aligned to the largest of
them, cut off 13 bits below its power of two (measured: a product of 2^3 is
kept beside one of 2^16, one of 2^2 is not): up to 7 2^-13 of the eight's
largest, for every eight of k; the sums of eights are fp32."""
from __future__ import annotations

import math

import torch

F = 2.0 ** -23
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FLOOR = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z / (1 + torch.exp(-z))


def slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    p = 1 / (1 + torch.exp(-z))
    return p * (1 + z * (1 - p))


def stored(value, dtype):
    return UNIT[dtype] * value.abs() + FLOOR[dtype]


def pre(x, w, bias, xs=None, ws=None):
    """z and its bound before any store."""
    x, w = x.double(), w.double()
    z, s = x @ w.t().contiguous(), x.abs() @ w.abs().t().contiguous()
    cut = 0.0
    if xs is not None:
        k = xs.double()[:, None] * ws.double()
        cut = 7 * 2.0 ** -13 * largest_of_eights(x, w) * k
        z, s = z * k, s * k
    if bias is not None:
        z, s = z + bias.double(), s + bias.double().abs()
    return z, (x.shape[1] + 8) * F * s + cut


def largest_of_eights(x, w):
    """Sum over k's eights of the largest |x w| among them."""
    x, w = x.abs().float(), w.abs().float()
    total = torch.zeros(len(x), len(w), dtype=torch.float64, device=x.device)
    for k in range(0, x.shape[1], 8):
        top = torch.zeros(len(x), len(w), device=x.device)
        for i in range(k, min(k + 8, x.shape[1])):
            top = torch.maximum(top, torch.outer(x[:, i], w[:, i]))
        total += top
    return total


def act_bound(z, ez):
    return 1.13 * ez + (8 * F + 2e-7) * z.abs()


def linear(x, w, bias, name, residual, dtype, xs=None, ws=None):
    """(y, bound)."""
    z, ez = pre(x, w, bias, xs, ws)
    y, e = act(name, z), act_bound(z, ez)
    if residual is not None:
        y = y + residual.double()
        e = e + 2 * F * y.abs()
    return y, e + stored(y.abs() + e, dtype)


def gated(x, w, bias, name, dtype, xs=None, ws=None):
    z, ez = pre(x, w, bias, xs, ws)
    (g, u), (eg, eu) = z.chunk(2, -1), ez.chunk(2, -1)
    a, ea = act(name, g), act_bound(g, eg)
    h = a * u
    e = ea * u.abs() + a.abs() * eu + ea * eu + 2 * F * h.abs()
    return h, e + stored(h.abs() + e, dtype)


def grads(dy, x, w, z, name, is_gated, dtype):
    """((dx, bound), (dw, bound), (db, bound))."""
    dy, x, w, z = dy.double(), x.double(), w.double(), (None if z is None else z.double())
    if is_gated:
        g, u = z.chunk(2, -1)
        d = torch.cat([dy * u * slope(name, g), dy * act(name, g)], -1)
        e = torch.cat([dy.abs() * u.abs() * 2e-6 * (1 + g.abs()),
                       dy.abs() * (8 * F + 2e-7) * g.abs()], -1)
    elif z is None:
        d, e = dy, torch.zeros_like(dy)
    else:
        d, e = dy * slope(name, z), dy.abs() * 2e-6 * (1 + z.abs())
    e = e + 4 * F * d.abs()
    q = e + stored(d.abs() + e, dtype)          # dz as the products read it
    m = d.abs() + q
    dx, dw, db = d @ w, d.t().contiguous() @ x, d.sum(0)
    ex = q @ w.abs() + (w.shape[0] + 8) * F * (m @ w.abs())
    ew = q.t().contiguous() @ x.abs() + (len(x) + 8) * F * (m.t().contiguous() @ x.abs())
    eb = e.sum(0) + (len(x) + 8) * F * m.sum(0)
    return tuple((v, b + stored(v.abs() + b, dtype)) for v, b in ((dx, ex), (dw, ew), (db, eb)))


def norm(x, residual, weight, eps, x_type):
    """(y, its bound before the store, s, its bound, rstd)."""
    s = x.double() if residual is None else x.double() + residual.double()
    r = torch.rsqrt((s * s).mean(-1, keepdim=True) + eps)
    y = s * r if weight is None else s * r * weight.double()
    return y, (s.shape[-1] + 16) * F * y.abs(), s, stored(s, x_type) + F * s.abs(), r[..., 0]


def norm_grads(dy, s, weight, rstd, dstream, s_type, w_type):
    """((ds, bound), (dw, bound))."""
    dy, s, r = dy.double(), s.double(), rstd.double()[:, None]
    n = s * r
    a = dy if weight is None else dy * weight.double()
    ds = r * (a - n * (a * n).mean(-1, keepdim=True))
    e = (s.shape[1] + 16) * F * r * (a.abs() + n.abs() * (a * n).abs().mean(-1, keepdim=True))
    if dstream is not None:
        ds = ds + dstream.double()
        e = e + F * ds.abs()
    dw = (dy * n).sum(0)
    ew = (len(s) + 16) * F * (dy * n).abs().sum(0)
    return (ds, e + stored(ds.abs() + e, s_type)), (dw, ew + stored(dw.abs() + ew, w_type))
