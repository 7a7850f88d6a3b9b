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

Where autograd records (a tensor requires a gradient and gradients are enabled)
add_rms_norm, linear and gated are recorded with these gradients; float8 and
`out` then raise.  They are differentiable once.

Errors raise RuntimeError with the "ffn ops: " prefix.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

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


# At a few rows the kernels take less time than a call's checks: the usual call
# runs in C (csrc/ffn_call.cpp), which returns None for any other, and the
# checks below take the cheapest queries.
@lru_cache(maxsize=None)
def _call():
    module = _lib.load_ffn_call()
    module.setup(torch.float16, torch.bfloat16, torch.float32, torch.uint8, _ACTS, _device,
                 _stream, torch.is_grad_enabled)
    return module


_VALUES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_HALVES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_OPERANDS = {**_HALVES, torch.float8_e4m3fn: _lib.E4M3}
_F32 = torch.float32
_MOST = 2 ** 31 - 1  # what the C entry points' sizes hold


def _rows(op: str, name: str, t):
    """(rows, columns, elements from row to row) of a tensor whose leading
    dimensions collapse to evenly spaced rows."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 2:
        rows, cols = shape
        step = stride[0]
    elif not shape:
        _fail(f"{op}: {name} must have at least one dimension")
    else:
        cols = shape[-1]
        rows, step = 1, cols
        for n, s in zip(reversed(shape[:-1]), reversed(stride[:-1])):
            if n == 0:  # no rows, whatever the others' spacing
                rows = 0
                break
            if n == 1:
                continue
            if rows == 1:
                step = s
            elif s != step * rows:
                _fail(f"{op}: {name}'s leading dimensions must collapse to evenly spaced rows")
            rows *= n
    if rows > _MOST or cols > _MOST:
        _fail(f"{op}: {name} has {rows} rows of {cols}, more than {_MOST} of either")
    if cols > 1 and stride[-1] != 1:
        _fail(f"{op}: {name}'s last dimension must be contiguous")
    # one row (or none) may be any distance from the next
    return rows, cols, (step if rows > 1 else cols)


def _index(op: str, t) -> int:
    if not t.is_cuda:
        _fail(f"{op}: tensors must be on a HIP device")
    return t.get_device()


def _type(op: str, name: str, dtype, allowed) -> int:
    kind = allowed.get(dtype)
    if kind is None:
        _fail(f"{op}: {name} is {dtype}, expected one of " + ", ".join(str(d) for d in allowed))
    return kind


def _vector(op: str, name: str, t, index: int, n: int, *allowed):
    """(address, type) of a contiguous vector of n on the operands' device."""
    if t.dtype not in allowed:
        _fail(f"{op}: {name} is {t.dtype}, expected one of " + ", ".join(str(d) for d in allowed))
    if t.numel() != n or not t.is_contiguous():
        _fail(f"{op}: {name} must be a contiguous tensor of {n} elements, got {tuple(t.shape)}")
    if t.get_device() != index:
        _fail(f"{op}: {name} must be on the same device as the others")
    return t.data_ptr(), _TYPES[t.dtype]


def _same(op: str, name: str, t, index: int, shape, dtype):
    """(address, row step) of t, which must have this shape, type and device."""
    if t.shape != shape:
        _fail(f"{op}: {name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        _fail(f"{op}: {name} is {t.dtype}, expected {dtype}")
    if t.get_device() != index:
        _fail(f"{op}: {name} must be on the same device as the others")
    return t.data_ptr(), _rows(op, name, t)[2]


def _launch(op: str, index: int, fn, *args) -> None:
    """fn(*args, stream) on the current stream of device `index`, with that
    device current; raises on a refusal."""
    if _device() == index:
        status = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _stream(index))
    if status != _lib.OK:
        _fail(f"{op}: {_lib.ffn_last_error()} (status {status})")


_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


def _space(n: int, like):
    """n bytes of workspace on like's device (None for none) and its address."""
    if n <= 0:
        return None, 0
    t = torch.empty(n, dtype=torch.uint8, device=like.device)
    return t, t.data_ptr()


def _recorded(*tensors) -> bool:
    """Whether autograd is to record a call on these (some may be None)."""
    for t in tensors:
        if t is not None and t.requires_grad:
            return torch.is_grad_enabled()
    return False


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
    if not save:
        done = _call().norm(x, residual, weight, eps, dtype)
        if done is not None:
            return Norm(done[0], None, done[1], None)
    if _recorded(x, residual, weight):
        if dtype == torch.float8_e4m3fn:
            _fail("add_rms_norm: float8 output has no gradient: call it under torch.no_grad()")
        y, rstd, *stream = _RecordedNorm.apply(eps, dtype, x, residual, weight)
        return Norm(y, None, stream[0] if stream else x, rstd if save else None)
    return _norm(x, residual, weight, eps, dtype, save)


def _norm(x, residual, weight, eps, dtype, save) -> Norm:
    op = "add_rms_norm"
    index, xd = _index(op, x), x.dtype
    xt = _type(op, "x", xd, _VALUES)
    rows, cols, ldx = _rows(op, "x", x)
    shape = x.shape
    wp = wt = rp = ldr = sp = cp = dp = 0
    scale = rstd = None
    stream = x
    if weight is not None:
        wp, wt = _vector(op, "weight", weight, index, cols, _F32, xd)
    if residual is not None:
        rp, ldr = _same(op, "residual", residual, index, shape, xd)
        stream = x.new_empty(shape)
        sp = stream.data_ptr()
    if dtype is None or dtype == xd:
        yt, y = xt, x.new_empty(shape)
    else:
        yt, y = _TYPES.get(dtype, -1), x.new_empty(shape, dtype=dtype)
        if yt == _lib.E4M3:
            scale = x.new_empty(shape[:-1], dtype=_F32)
            cp = scale.data_ptr()
    if save:
        rstd = x.new_empty(shape[:-1], dtype=_F32)
        dp = rstd.data_ptr()
    _launch(op, index, _lib.load_ffn().bvml_ffn_add_rms_norm, x.data_ptr(), ldx, rp, ldr, wp, rows,
            cols, eps, xt, wt, yt, y.data_ptr(), cols, sp, cols, cp, dp)
    return Norm(y, scale, stream, rstd)


class _RecordedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, eps, dtype, x, residual, weight):
        n = _norm(x, residual, weight, eps, dtype, True)
        ctx.save_for_backward(n.stream, weight, n.rstd)
        ctx.y_shape, ctx.y_type = n.y.shape, n.y.dtype
        ctx.mark_non_differentiable(n.rstd)
        ctx.set_materialize_grads(False)
        return (n.y, n.rstd) if residual is None else (n.y, n.rstd, n.stream)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _, dstream=None):
        stream, weight, rstd = ctx.saved_tensors
        dy = stream.new_zeros(ctx.y_shape, dtype=ctx.y_type) if dy is None else dy.contiguous()
        ds, dw = add_rms_norm_backward(dy, stream, weight, rstd,
                                       None if dstream is None else dstream.contiguous(),
                                       need_weight=ctx.needs_input_grad[4])
        return None, None, ds, ds if ctx.needs_input_grad[3] else None, dw


def add_rms_norm_backward(dy, stream, weight, rstd, dstream=None, *, need_weight: bool = True):
    """(ds, dweight): the gradient of x and of residual, both ds, and the
    weight's, from dy, the forward pass's stream and rstd, and the gradient
    that reaches the stream itself."""
    op = "add_rms_norm_backward"
    index, sd = _index(op, stream), stream.dtype
    st = _type(op, "stream", sd, _VALUES)
    dt = _type(op, "dy", dy.dtype, _VALUES)
    rows, cols, lds = _rows(op, "stream", stream)
    yp, lddy = _same(op, "dy", dy, index, stream.shape, dy.dtype)
    rp, _ = _vector(op, "rstd", rstd, index, rows, _F32)
    wp = wt = gp = ldg = dwp = n = 0
    dw = None
    lib = _lib.load_ffn()
    if weight is not None:
        wp, wt = _vector(op, "weight", weight, index, cols, _F32, sd)
        if need_weight:
            dw = torch.empty_like(weight)
            dwp = dw.data_ptr()
            n = lib.bvml_ffn_add_rms_norm_backward_workspace(rows, cols)
    if dstream is not None:
        gp, ldg = _same(op, "dstream", dstream, index, stream.shape, sd)
    ds = stream.new_empty(stream.shape)
    space, sp = _space(n, stream)
    _launch(op, index, lib.bvml_ffn_add_rms_norm_backward, yp, lddy, stream.data_ptr(), lds, wp, rp,
            gp, ldg, rows, cols, dt, st, wt, ds.data_ptr(), cols, dwp, sp, n)
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
    index, xd = _index(op, x), x.dtype
    kind = _type(op, "x", xd, _OPERANDS)
    if w.dtype != xd:
        _fail(f"{op}: w is {w.dtype}, x {xd}: one type for both")
    if w.dim() != 2:
        _fail(f"{op}: w must have two dimensions")
    if w.get_device() != index:
        _fail(f"{op}: w must be on the same device as the others")
    M, K, ldx = _rows(op, "x", x)
    R, Kw, ldw = _rows(op, "w", w)
    if Kw != K:
        _fail(f"{op}: w has rows of {Kw}, x of {K}")
    N = R
    if gated:
        if R % 2:
            _fail(f"{op}: w must stack the gate's and the other half's rows: {R} is odd")
        N = R // 2
    code = _ACTS.get(act)
    if code is None:
        _fail(f"{op}: unknown activation {act!r}, expected one of " + ", ".join(_ACTS))
    if dtype is None or dtype == xd:
        dtype = torch.bfloat16 if kind == _lib.E4M3 else xd
    yt = _type(op, "the output", dtype, _VALUES)
    bp = bt = xs = ws = rp = ldr = zp = 0
    z = None
    if bias is not None:
        bp, bt = _vector(op, "bias", bias, index, R, dtype, _F32, xd)
    if x_scale is not None:
        xs, _ = _vector(op, "x_scale", x_scale, index, M, _F32)
    if w_scale is not None:
        ws, _ = _vector(op, "w_scale", w_scale, index, R, _F32)
    shape = (M, N) if x.dim() == 2 else (*x.shape[:-1], N)
    if out is None:
        out = x.new_empty(shape) if dtype == xd else x.new_empty(shape, dtype=dtype)
        yp, ldy = out.data_ptr(), N
    else:
        yp, ldy = _same(op, "out", out, index, shape, dtype)
    if residual is not None:
        rp, ldr = _same(op, "residual", residual, index, shape, dtype)
    if save:
        z = x.new_empty((*shape[:-1], R))
        zp = z.data_ptr()
    n = _forward_space(gated, M, N, K, kind)
    space, sp = _space(n, x)
    lib = _lib.load_ffn()
    if gated:
        _launch(op, index, lib.bvml_ffn_gated, x.data_ptr(), ldx, w.data_ptr(), ldw, bp, xs, ws, M,
                N, K, kind, yt, bt, code, yp, ldy, zp, R, sp, n)
    else:
        _launch(op, index, lib.bvml_ffn_linear, x.data_ptr(), ldx, w.data_ptr(), ldw, bp, xs, ws,
                rp, ldr, M, N, K, kind, yt, bt, code, yp, ldy, zp, R, sp, n)
    return Product(out, z)


def linear(x, w, bias=None, act: str = "none", residual=None, *, x_scale=None, w_scale=None,
           dtype=None, save: bool = False, out=None) -> Product:
    """y = act(x w^T + bias) + residual for x (..., K) and w (N, K), float16 or
    bfloat16, or both float8_e4m3fn with x_scale (one a row of x) and w_scale
    (one a row of w).  act: none, relu, gelu, gelu_tanh or silu.  `dtype`: the
    output's (and the residual's), x's type or float32 (from float8: bfloat16
    by default, or float16 or float32).  `out` may be `residual` itself.
    Returns Product(y, z): z the pre-activations in x's type, with save."""
    if x_scale is None and w_scale is None and not save and out is None:
        y = _call().product(x, w, bias, act, residual, False, dtype)
        if y is not None:
            return Product(y, None)
    return _product("linear", False, x, w, bias, act, residual, x_scale, w_scale, dtype, save, out)


def gated(x, w, bias=None, act: str = "silu", *, x_scale=None, w_scale=None, dtype=None,
          save: bool = False, out=None) -> Product:
    """h = act(x wg^T + bg) * (x wu^T + bu) for x (..., K) and w = [wg; wu]
    (2N, K), in one kernel; types as linear.  Returns Product(h, z): z (..., 2N)
    the pre-activations of both halves, with save."""
    if x_scale is None and w_scale is None and not save and out is None:
        y = _call().product(x, w, bias, act, None, True, dtype)
        if y is not None:
            return Product(y, None)
    return _product("gated", True, x, w, bias, act, None, x_scale, w_scale, dtype, save, out)


def _product(op: str, gated: bool, x, w, bias, act, residual, x_scale, w_scale, dtype, save, out):
    if not _recorded(x, w, bias, residual, x_scale, w_scale, out):
        return _forward(op, gated, x, w, bias, act, residual, x_scale, w_scale, dtype, save, out)
    if x.dtype == torch.float8_e4m3fn or x_scale is not None or w_scale is not None:
        _fail(f"{op}: float8 operands have no gradient: call it under torch.no_grad()")
    if out is not None:
        _fail(f"{op}: a given output has no gradient: call it under torch.no_grad()")
    return Product(*_RecordedProduct.apply(op, gated, act, dtype, save, x, w, bias, residual))


class _RecordedProduct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, op, gated, act, dtype, save, x, w, bias, residual):
        sloped = gated or act != "none"
        y, z = _forward(op, gated, x, w, bias, act, residual, None, None, dtype, save or sloped,
                        None)
        ctx.save_for_backward(x, w, z if sloped else None)
        ctx.call, ctx.bias = (op + "_backward", gated), bias is not None and (bias.shape, bias.dtype)
        ctx.act = act
        if not save:
            return y, None
        ctx.mark_non_differentiable(z)
        return y, z

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _):
        x, w, z = ctx.saved_tensors
        need_x, need_w, need_bias, need_residual = ctx.needs_input_grad[5:]
        op, gated = ctx.call
        dx, dw, db = _backward(op, gated, dy.contiguous(), x, w, z, ctx.act, need_x, need_w,
                               need_bias)
        if need_bias:
            shape, dtype = ctx.bias
            db = db.reshape(shape).to(dtype)
        return None, None, None, None, None, dx, dw, db, dy if need_residual else None


def _backward(op: str, is_gated: bool, dy, x, w, z, act, need_x, need_w, need_bias):
    index, xd = _index(op, x), x.dtype
    kind = _type(op, "x", xd, _HALVES)
    if dy.dtype != xd and dy.dtype != _F32:
        _fail(f"{op}: the output's gradient is {dy.dtype}, expected {xd} or float32")
    if w.dtype != xd or w.dim() != 2 or w.get_device() != index:
        _fail(f"{op}: w must be a matrix of x's type on its device")
    M, K, ldx = _rows(op, "x", x)
    R, Kw, ldw = _rows(op, "w", w)
    if Kw != K or (is_gated and R % 2):
        _fail(f"{op}: w is {tuple(w.shape)}, x has rows of {K}")
    N = R // 2 if is_gated else R
    code = _ACTS.get(act)
    if code is None:
        _fail(f"{op}: unknown activation {act!r}, expected one of " + ", ".join(_ACTS))
    lead = x.shape[:-1]
    yp, lddy = _same(op, "dy", dy, index, (*lead, N), dy.dtype)
    zp, ldz = 0, R
    if z is not None:
        zp, ldz = _same(op, "z", z, index, (*lead, R), xd)
    elif is_gated or act != "none":
        _fail(f"{op}: the pre-activations z are needed (forward with save=True)")
    dx = x.new_empty(x.shape) if need_x else None
    dw = x.new_empty((R, K)) if need_w else None
    db = x.new_empty((R,)) if need_bias else None
    n = _backward_space(is_gated, M, N, K)
    space, sp = _space(n, x)
    lib = _lib.load_ffn()
    _launch(op, index, lib.bvml_ffn_gated_backward if is_gated else lib.bvml_ffn_linear_backward,
            yp, lddy, x.data_ptr(), ldx, w.data_ptr(), ldw, zp, ldz, M, N, K, kind,
            _TYPES[dy.dtype], code, 0 if dx is None else dx.data_ptr(), K,
            0 if dw is None else dw.data_ptr(), K, 0 if db is None else db.data_ptr(), sp, n)
    return dx, dw, db


def linear_backward(dy, x, w, z=None, act: str = "none", *, need_x: bool = True,
                    need_w: bool = True, need_bias: bool = True):
    """(dx, dw, dbias) of linear, in x's type, from dy (x's type or float32),
    its inputs and its saved z (not needed with act "none"); None for those
    not needed.  The residual's gradient is dy itself.  The products take
    dz = dy act'(z) in x's type: with float16 a float32 dy, too, is cut to its
    range."""
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
