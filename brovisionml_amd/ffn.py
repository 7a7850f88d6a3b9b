"""The feed-forward half of a pre-norm transformer block on HIP device tensors:
the operators of include/bvml_ffn.h, forward and backward.

  add_rms_norm(x, residual, weight, eps)     s = x + residual,
                                             y = s / sqrt(mean(s^2) + eps) * weight
  linear(x, w, bias, act, residual)          y = act(x w^T + bias) + residual
  gated(x, w, bias, act)                     h = act(x wg^T + bg) * (x wu^T + bu)

with w = [wg; wu] stacked, and add_rms_norm_backward, linear_backward and
gated_backward for their gradients.  FeedForward strings them together.

Tensors are torch tensors on one HIP device (torch is the allocator and stream
provider), the last dimension contiguous, the others collapsing to rows a
fixed distance apart.  float16, bfloat16 and, for the norm, float32; the
products also take float8_e4m3fn operands with a float32 scale a row, as
add_rms_norm(dtype=torch.float8_e4m3fn) leaves them.  Every call is
asynchronous on the current stream of the tensors' device.

Errors raise RuntimeError with the "ffn ops: " prefix.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from . import _lib
from .dsine import _launch

_WHO = "ffn ops: "
_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16,
          torch.float8_e4m3fn: _lib.E4M3}
_ACTS = _lib.ACTS


class Norm(NamedTuple):
    """add_rms_norm's results; scale with float8 y, rstd with save."""
    y: torch.Tensor
    scale: Optional[torch.Tensor]
    stream: torch.Tensor
    rstd: Optional[torch.Tensor]


class Product(NamedTuple):
    """linear's and gated's results; z, the pre-activations, with save."""
    y: torch.Tensor
    z: Optional[torch.Tensor]


def _fail(msg: str):
    raise RuntimeError(_WHO + msg)


def _raise_status(op: str, status: int) -> None:
    if status != _lib.OK:
        _fail(f"{op}: {_lib.ffn_last_error()} (status {status})")


def _rows(op: str, name: str, t):
    """(rows, columns, elements from row to row) of a tensor whose leading
    dimensions collapse to evenly spaced rows."""
    shape, stride = t.shape, t.stride()
    if not shape:
        _fail(f"{op}: {name} must have at least one dimension")
    cols = shape[-1]
    if len(shape) == 2:
        rows, step = shape[0], stride[0]
    else:
        rows, step = 1, cols
        for n, s in zip(reversed(shape[:-1]), reversed(stride[:-1])):
            if n == 1:
                continue
            if rows == 1:
                step = s
            elif s != step * rows:
                _fail(f"{op}: {name}'s leading dimensions must collapse to evenly spaced rows")
            rows *= n
    if cols > 1 and stride[-1] != 1:
        _fail(f"{op}: {name}'s last dimension must be contiguous")
    # one row (or none) may be any distance from the next
    return rows, cols, (step if rows > 1 else cols)


def _check(op: str, first, **tensors) -> None:
    """Every tensor on one HIP device."""
    if not first.is_cuda:
        _fail(f"{op}: tensors must be on a HIP device")
    index = first.get_device()
    for name, t in tensors.items():
        if t is not None and t.get_device() != index:
            _fail(f"{op}: {name} must be on the same device as the others")


def _type(op: str, name: str, dtype, allowed) -> int:
    if dtype not in allowed:
        _fail(f"{op}: {name} is {dtype}, expected one of "
              + ", ".join(str(d) for d in allowed))
    return _TYPES[dtype]


def _vector(op: str, name: str, t, n: int, allowed):
    """(address, type) of a contiguous vector of n, (0, F32) for None."""
    if t is None:
        return 0, _lib.F32
    kind = _type(op, name, t.dtype, allowed)
    if t.numel() != n or not t.is_contiguous():
        _fail(f"{op}: {name} must be a contiguous tensor of {n} elements, got {tuple(t.shape)}")
    return t.data_ptr(), kind


_VALUES = (torch.float32, torch.float16, torch.bfloat16)
_HALVES = (torch.float16, torch.bfloat16)
_F32 = (torch.float32,)


def _same(op: str, name: str, t, shape, dtype):
    """Row step of t, which must have this shape and type."""
    if t.shape != shape:
        _fail(f"{op}: {name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        _fail(f"{op}: {name} is {t.dtype}, expected {dtype}")
    return _rows(op, name, t)[2]


def _space(n: int, like):
    """n bytes of workspace on like's device (None for none) and its address."""
    if n == 0:
        return None, 0
    t = torch.empty(n, dtype=torch.uint8, device=like.device)
    return t, t.data_ptr()


# ---------------------------------------------------------------------------
# the norm
# ---------------------------------------------------------------------------
def add_rms_norm(x, residual=None, weight=None, eps: float = 1e-6, *, dtype=None,
                 save: bool = False) -> Norm:
    """s = x + residual and y = s / sqrt(mean(s^2) + eps) * weight over the last
    dimension.  Returns Norm: y in `dtype` (x's by default; float16 or
    bfloat16 from float32; float8_e4m3fn with `scale`, one a row, so that
    y = q * scale), `stream` = s in x's type (x itself without a residual) and,
    with save, the rows' rstd for the backward pass.  The weight is float32
    or of x's type; None means ones."""
    op = "add_rms_norm"
    _check(op, x, residual=residual, weight=weight)
    xt = _type(op, "x", x.dtype, _VALUES)
    rows, cols, ldx = _rows(op, "x", x)
    ldr = 0 if residual is None else _same(op, "residual", residual, x.shape, x.dtype)
    wp, wt = _vector(op, "weight", weight, cols, (torch.float32, x.dtype))
    dtype = x.dtype if dtype is None else dtype
    yt = _TYPES.get(dtype, -1)
    y = torch.empty(x.shape, dtype=dtype, device=x.device)
    lead = x.shape[:-1]
    scale = torch.empty(lead, dtype=torch.float32, device=x.device) if yt == _lib.E4M3 else None
    rstd = torch.empty(lead, dtype=torch.float32, device=x.device) if save else None
    stream = x if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    st = _launch(x, _lib.load_ffn().bvml_ffn_add_rms_norm, x.data_ptr(), ldx,
                 0 if residual is None else residual.data_ptr(), ldr, wp, rows, cols, eps, xt, wt,
                 yt, y.data_ptr(), cols, 0 if residual is None else stream.data_ptr(), cols,
                 0 if scale is None else scale.data_ptr(), 0 if rstd is None else rstd.data_ptr())
    _raise_status(op, st)
    return Norm(y, scale, stream, rstd)


def add_rms_norm_backward(dy, stream, weight, rstd, dstream=None, *, need_weight: bool = True):
    """(ds, dweight): the gradient of x and of residual, both ds, and the
    weight's, from dy, the forward pass's stream and rstd, and the gradient
    that reaches the stream itself."""
    op = "add_rms_norm_backward"
    _check(op, stream, dy=dy, weight=weight, rstd=rstd, dstream=dstream)
    st_t = _type(op, "stream", stream.dtype, _VALUES)
    dt = _type(op, "dy", dy.dtype, _VALUES)
    rows, cols, lds = _rows(op, "stream", stream)
    lddy = _same(op, "dy", dy, stream.shape, dy.dtype)
    lddst = 0 if dstream is None else _same(op, "dstream", dstream, stream.shape, stream.dtype)
    wp, wt = _vector(op, "weight", weight, cols, (torch.float32, stream.dtype))
    rp, _ = _vector(op, "rstd", rstd, rows, _F32)
    ds = torch.empty(stream.shape, dtype=stream.dtype, device=stream.device)
    dw = torch.empty_like(weight) if weight is not None and need_weight else None
    lib = _lib.load_ffn()
    n = lib.bvml_ffn_add_rms_norm_backward_workspace(rows, cols) if dw is not None else 0
    space, sp = _space(max(n, 0), stream)
    st = _launch(stream, lib.bvml_ffn_add_rms_norm_backward, dy.data_ptr(), lddy,
                 stream.data_ptr(), lds, wp, rp, 0 if dstream is None else dstream.data_ptr(),
                 lddst, rows, cols, dt, st_t, wt, ds.data_ptr(), cols,
                 0 if dw is None else dw.data_ptr(), sp, n)
    _raise_status(op, st)
    return ds, dw


# ---------------------------------------------------------------------------
# the products
# ---------------------------------------------------------------------------
@lru_cache(maxsize=4096)
def _forward_space(gated: bool, M: int, N: int, K: int, kind: int) -> int:
    lib = _lib.load_ffn()
    return (lib.bvml_ffn_gated_workspace if gated else lib.bvml_ffn_linear_workspace)(M, N, K, kind)


@lru_cache(maxsize=4096)
def _backward_space(gated: bool, M: int, N: int, K: int) -> int:
    lib = _lib.load_ffn()
    return (lib.bvml_ffn_gated_backward_workspace if gated
            else lib.bvml_ffn_linear_backward_workspace)(M, N, K)


def _forward(op: str, gated: bool, x, w, bias, act, residual, x_scale, w_scale, dtype, save, out):
    _check(op, x, w=w, bias=bias, residual=residual, x_scale=x_scale, w_scale=w_scale, out=out)
    kind = _type(op, "x", x.dtype, (*_HALVES, torch.float8_e4m3fn))
    if w.dtype != x.dtype:
        _fail(f"{op}: w is {w.dtype}, x {x.dtype}: one type for both")
    if w.dim() != 2:
        _fail(f"{op}: w must have two dimensions")
    M, K, ldx = _rows(op, "x", x)
    R, Kw, ldw = _rows(op, "w", w)
    if Kw != K:
        _fail(f"{op}: w has rows of {Kw}, x of {K}")
    if gated and R % 2:
        _fail(f"{op}: w must stack the gate's and the other half's rows: {R} is odd")
    N = R // 2 if gated else R
    if act not in _ACTS:
        _fail(f"{op}: unknown activation {act!r}, expected one of " + ", ".join(_ACTS))
    e4m3 = kind == _lib.E4M3
    if dtype is None:
        dtype = torch.bfloat16 if e4m3 else x.dtype
    yt = _TYPES.get(dtype, -1)
    if yt not in (_lib.F32, _lib.F16, _lib.BF16):
        _fail(f"{op}: the output cannot be {dtype}")
    bp, bt = _vector(op, "bias", bias, R, (torch.float32, dtype, x.dtype))
    xs, _ = _vector(op, "x_scale", x_scale, M, _F32)
    ws, _ = _vector(op, "w_scale", w_scale, R, _F32)
    shape = (*x.shape[:-1], N)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=x.device)
        ldy = N
    else:
        ldy = _same(op, "out", out, shape, dtype)
    rp, ldr = 0, 0
    if residual is not None:
        ldr = _same(op, "residual", residual, shape, dtype)
        rp = residual.data_ptr()
    z, zp = None, 0
    if save:
        z = torch.empty((*x.shape[:-1], R), dtype=x.dtype, device=x.device)
        zp = z.data_ptr()
    n = _forward_space(gated, M, N, K, kind) if M else 0
    space, sp = _space(max(n, 0), x)
    lib = _lib.load_ffn()
    if gated:
        st = _launch(x, lib.bvml_ffn_gated, x.data_ptr(), ldx, w.data_ptr(), ldw, bp, xs, ws, M, N,
                     K, kind, yt, bt, _ACTS[act], out.data_ptr(), ldy, zp, R, sp, n)
    else:
        st = _launch(x, lib.bvml_ffn_linear, x.data_ptr(), ldx, w.data_ptr(), ldw, bp, xs, ws, rp,
                     ldr, M, N, K, kind, yt, bt, _ACTS[act], out.data_ptr(), ldy, zp, R, sp, n)
    _raise_status(op, st)
    return Product(out, z)


def linear(x, w, bias=None, act: str = "none", residual=None, *, x_scale=None, w_scale=None,
           dtype=None, save: bool = False, out=None) -> Product:
    """y = act(x w^T + bias) + residual for x (..., K) and w (N, K), float16 or
    bfloat16, or both float8_e4m3fn with x_scale (one a row of x) and w_scale
    (one a row of w).  act: none, relu, gelu, gelu_tanh or silu.  `dtype`: the
    output's (and the residual's), x's type or float32 (from float8: bfloat16
    by default, or float16 or float32).  `out` may be `residual` itself.
    Returns Product(y, z): z the pre-activations in x's type, with save."""
    return _forward("linear", False, x, w, bias, act, residual, x_scale, w_scale, dtype, save, out)


def gated(x, w, bias=None, act: str = "silu", *, x_scale=None, w_scale=None, dtype=None,
          save: bool = False, out=None) -> Product:
    """h = act(x wg^T + bg) * (x wu^T + bu) for x (..., K) and w = [wg; wu]
    (2N, K), in one kernel; types as linear.  Returns Product(h, z): z (..., 2N)
    the pre-activations of both halves, with save."""
    return _forward("gated", True, x, w, bias, act, None, x_scale, w_scale, dtype, save, out)


def _backward(op: str, is_gated: bool, dy, x, w, z, act, need_x, need_w, need_bias):
    _check(op, dy, x=x, w=w, z=z)
    kind = _type(op, "x", x.dtype, _HALVES)
    dt = _type(op, "dy", dy.dtype, (torch.float32, x.dtype))
    if w.dtype != x.dtype or w.dim() != 2:
        _fail(f"{op}: w must be a matrix of x's type")
    M, K, ldx = _rows(op, "x", x)
    R, Kw, ldw = _rows(op, "w", w)
    if Kw != K or (is_gated and R % 2):
        _fail(f"{op}: w is {tuple(w.shape)}, x has rows of {K}")
    N = R // 2 if is_gated else R
    if act not in _ACTS:
        _fail(f"{op}: unknown activation {act!r}, expected one of " + ", ".join(_ACTS))
    lddy = _same(op, "dy", dy, (*x.shape[:-1], N), dy.dtype)
    zp, ldz = 0, R
    if z is not None:
        ldz = _same(op, "z", z, (*x.shape[:-1], R), x.dtype)
        zp = z.data_ptr()
    elif is_gated or act != "none":
        _fail(f"{op}: the pre-activations z are needed (forward with save=True)")
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
    dw = torch.empty((R, K), dtype=x.dtype, device=x.device) if need_w else None
    db = torch.empty(R, dtype=x.dtype, device=x.device) if need_bias else None
    n = _backward_space(is_gated, M, N, K)
    space, sp = _space(max(n, 0), x)
    lib = _lib.load_ffn()
    fn = lib.bvml_ffn_gated_backward if is_gated else lib.bvml_ffn_linear_backward
    st = _launch(x, fn, dy.data_ptr(), lddy, x.data_ptr(), ldx, w.data_ptr(), ldw, zp, ldz, M, N,
                 K, kind, dt, _ACTS[act], 0 if dx is None else dx.data_ptr(), K,
                 0 if dw is None else dw.data_ptr(), K, 0 if db is None else db.data_ptr(), sp, n)
    _raise_status(op, st)
    return dx, dw, db


def linear_backward(dy, x, w, z=None, act: str = "none", *, need_x: bool = True,
                    need_w: bool = True, need_bias: bool = True):
    """(dx, dw, dbias) of linear, in x's type, from dy (x's type or float32),
    its inputs and its saved z (not needed with act "none"); None for those
    not needed.  The residual's gradient is dy itself."""
    return _backward("linear_backward", False, dy, x, w, z, act, need_x, need_w, need_bias)


def gated_backward(dh, x, w, z, act: str = "silu", *, need_x: bool = True, need_w: bool = True,
                   need_bias: bool = True):
    """(dx, dw, dbias) of gated, in x's type, from dh, its inputs and its saved
    z; None for those not needed."""
    return _backward("gated_backward", True, dh, x, w, z, act, need_x, need_w, need_bias)


# ---------------------------------------------------------------------------
# the three together
# ---------------------------------------------------------------------------
class FeedForward:
    """The feed-forward half of a pre-norm transformer block,

        s = x + residual;  out = s + down(gated(norm(s)))

    on the operators above: norm_weight (K), w_in (2N, K) = [gate; up], w_out
    (K, N), biases optional, the products' type theirs; x, residual and the
    stream in that type or float32.  forward() returns the new stream;
    with save=True also what backward() takes."""

    def __init__(self, norm_weight, w_in, w_out, b_in=None, b_out=None, act: str = "silu",
                 eps: float = 1e-6):
        self.norm_weight, self.w_in, self.w_out = norm_weight, w_in, w_out
        self.b_in, self.b_out, self.act, self.eps = b_in, b_out, act, eps

    def forward(self, x, residual=None, *, save: bool = False):
        n = add_rms_norm(x, residual, self.norm_weight, self.eps, dtype=self.w_in.dtype, save=save)
        h = gated(n.y, self.w_in, self.b_in, self.act, save=save)
        out = linear(h.y, self.w_out, self.b_out, residual=n.stream, dtype=x.dtype).y
        return (out, (n, h)) if save else out

    def backward(self, dout, saved):
        """The gradients by name: x (and residual), norm_weight, w_in, w_out,
        and b_in, b_out where there are biases."""
        n, h = saved
        g = {}
        dh, g["w_out"], g["b_out"] = linear_backward(dout, h.y, self.w_out,
                                                     need_bias=self.b_out is not None)
        dy, g["w_in"], g["b_in"] = gated_backward(dh, n.y, self.w_in, h.z, self.act,
                                                  need_bias=self.b_in is not None)
        g["x"], g["norm_weight"] = add_rms_norm_backward(dy, n.stream, self.norm_weight, n.rstd,
                                                         dstream=dout)
        return {k: v for k, v in g.items() if v is not None}
