"""The feed-forward library without a GPU: it exports what include/bvml_ffn.h
declares and nothing else, refuses bad arguments before any launch (every call
here fails its checks or has nothing to do), and its launch plan reaches every
kernel at the sizes the GPU tests run."""
from __future__ import annotations

import os
import re
import subprocess
import sys

import pytest
import torch

from brovisionml_amd import _lib, ffn
from brovisionml_amd.build import INCLUDE, LIB_FFN

A = 0x10000000  # never dereferenced; arrays sit 16 MiB apart
STEP = 1 << 24
X, W, B, R, Y, Z, S, T, WORK = (A + STEP * i for i in range(9))


def test_exports_are_the_header():
    with open(os.path.join(INCLUDE, "bvml_ffn.h")) as f:
        declared = set(re.findall(r"\b(bvml_ffn_\w+)\s*\(", f.read()))
    assert sorted(declared) == sorted(_lib.FFN_EXPORTS)
    out = subprocess.run(["nm", "-D", "--defined-only", LIB_FFN], stdout=subprocess.PIPE, text=True,
                         check=True).stdout
    names = [ln.split()[-1] for ln in out.splitlines() if ln.split()[1] in "TDBRVWiu"]
    assert sorted(names) == sorted(declared)
    assert _lib.load_ffn().bvml_ffn_version().decode() == "0.1.0"


def norm(**kw):
    a = dict(x=X, ldx=64, residual=R, ldr=64, weight=B, rows=4, cols=64, eps=1e-6, xt=_lib.BF16,
             wt=_lib.BF16, yt=_lib.BF16, y=Y, ldy=64, stream=S, lds=64, scale=0, rstd=T, s=0)
    a.update(kw)
    return _lib.load_ffn().bvml_ffn_add_rms_norm(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), _lib.FFN_ESHAPE), (dict(cols=0), _lib.FFN_ESHAPE),
    (dict(ldx=63), _lib.FFN_ESHAPE), (dict(ldy=63), _lib.FFN_ESHAPE),
    (dict(lds=1), _lib.FFN_ESHAPE), (dict(cols=32769, ldx=40000), _lib.FFN_ESIZE),
    (dict(ldx=1 << 23), _lib.FFN_ESIZE), (dict(eps=-1.0), _lib.FFN_EPARAM),
    (dict(eps=float("nan")), _lib.FFN_EPARAM), (dict(x=0), _lib.FFN_ENULL),
    (dict(y=0), _lib.FFN_ENULL), (dict(xt=_lib.E4M3), _lib.FFN_ETYPE),
    (dict(xt=7), _lib.FFN_ETYPE), (dict(wt=_lib.F16), _lib.FFN_ETYPE),
    (dict(yt=_lib.F16), _lib.FFN_ETYPE), (dict(yt=_lib.F32), _lib.FFN_ETYPE),
    (dict(yt=_lib.E4M3), _lib.FFN_ENULL), (dict(scale=Z), _lib.FFN_ETYPE),
    (dict(y=X), _lib.FFN_EALIAS), (dict(y=R + 64), _lib.FFN_EALIAS),
    (dict(stream=X + 128), _lib.FFN_EALIAS), (dict(rstd=Y), _lib.FFN_EALIAS),
    (dict(stream=X, ldx=128, rows=2), _lib.FFN_EALIAS), (dict(rows=0, x=0, y=0), _lib.OK),
])
def test_norm_refuses(kw, code):
    assert norm(**kw) == code
    if code:
        assert _lib.ffn_last_error().startswith("add_rms_norm: ")


def norm_grad(**kw):
    a = dict(dy=X, lddy=64, s=R, lds=64, weight=B, rstd=T, dstream=S, ldds=64, rows=4, cols=64,
             dt=_lib.BF16, st=_lib.BF16, wt=_lib.BF16, ds=Y, ldy=64, dw=Z, work=WORK,
             bytes=1 << 20, stream=0)
    a.update(kw)
    return _lib.load_ffn().bvml_ffn_add_rms_norm_backward(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), _lib.FFN_ESHAPE), (dict(cols=0), _lib.FFN_ESHAPE),
    (dict(lddy=3), _lib.FFN_ESHAPE), (dict(cols=40000), _lib.FFN_ESIZE),
    (dict(st=_lib.E4M3), _lib.FFN_ETYPE), (dict(dt=_lib.E4M3), _lib.FFN_ETYPE),
    (dict(wt=_lib.F16), _lib.FFN_ETYPE), (dict(rstd=0), _lib.FFN_ENULL),
    (dict(dy=0), _lib.FFN_ENULL), (dict(ds=0), _lib.FFN_ENULL), (dict(ds=X), _lib.FFN_EALIAS),
    (dict(dw=B), _lib.FFN_EALIAS), (dict(work=0), _lib.FFN_EWORK),
    (dict(bytes=4), _lib.FFN_EWORK), (dict(work=Y), _lib.FFN_EALIAS),
])
def test_norm_backward_refuses(kw, code):
    assert norm_grad(**kw) == code
    assert _lib.ffn_last_error().startswith("add_rms_norm_backward: ")


def product(gated=False, **kw):
    a = dict(x=X, ldx=64, w=W, ldw=64, bias=B, xs=0, ws=0, residual=R, ldr=48, M=100, N=48, K=64,
             it=_lib.BF16, ot=_lib.BF16, bt=_lib.BF16, act=4, y=Y, ldy=48, z=Z, ldz=96, work=WORK,
             bytes=1 << 24, stream=0)
    a.update(kw)
    if gated:
        del a["residual"], a["ldr"]
    lib = _lib.load_ffn()
    return (lib.bvml_ffn_gated if gated else lib.bvml_ffn_linear)(*a.values())


REFUSED = [
    (dict(M=-1), _lib.FFN_ESHAPE), (dict(N=0), _lib.FFN_ESHAPE), (dict(K=0), _lib.FFN_ESHAPE),
    (dict(ldx=63), _lib.FFN_ESHAPE), (dict(ldw=1), _lib.FFN_ESHAPE),
    (dict(ldy=47), _lib.FFN_ESHAPE), (dict(ldz=47), _lib.FFN_ESHAPE),
    (dict(ldw=1 << 22), _lib.FFN_ESIZE), (dict(act=5), _lib.FFN_EPARAM),
    (dict(act=-1), _lib.FFN_EPARAM), (dict(x=0), _lib.FFN_ENULL), (dict(w=0), _lib.FFN_ENULL),
    (dict(y=0), _lib.FFN_ENULL), (dict(it=_lib.F32), _lib.FFN_ETYPE),
    (dict(ot=_lib.F16), _lib.FFN_ETYPE), (dict(ot=_lib.E4M3), _lib.FFN_ETYPE),
    (dict(bt=_lib.F16), _lib.FFN_ETYPE), (dict(it=_lib.E4M3), _lib.FFN_ENULL),
    (dict(xs=S, ws=T), _lib.FFN_ETYPE), (dict(it=_lib.E4M3, xs=S, ws=T), _lib.FFN_ETYPE),
    (dict(it=_lib.E4M3, xs=S, z=0), _lib.FFN_ENULL), (dict(y=X), _lib.FFN_EALIAS),
    (dict(y=W + 2), _lib.FFN_EALIAS), (dict(z=Y), _lib.FFN_EALIAS),
    (dict(y=B), _lib.FFN_EALIAS),
]


@pytest.mark.parametrize("kw,code", REFUSED + [
    (dict(residual=Y + 2), _lib.FFN_EALIAS), (dict(residual=Y, ldr=50), _lib.FFN_EALIAS),
    (dict(ldr=3), _lib.FFN_ESHAPE),
    # a split sum needs its workspace
    (dict(M=128, N=64, K=8192, ldx=8192, ldw=8192, ldy=64, ldr=64, z=0, work=0), _lib.FFN_EWORK),
    (dict(M=128, N=64, K=8192, ldx=8192, ldw=8192, ldy=64, ldr=64, z=0, bytes=64),
     _lib.FFN_EWORK)])
def test_linear_refuses(kw, code):
    assert product(**kw) == code
    assert _lib.ffn_last_error().startswith("linear: ")


@pytest.mark.parametrize("kw,code", REFUSED + [(dict(ldz=95), _lib.FFN_ESHAPE),
                                               (dict(N=1 << 30), _lib.FFN_ESIZE)])
def test_gated_refuses(kw, code):
    assert product(gated=True, **kw) == code
    assert _lib.ffn_last_error().startswith("gated: ")


def grads(gated=False, **kw):
    a = dict(dy=Y, lddy=48, x=X, ldx=64, w=W, ldw=64, z=Z, ldz=96, M=100, N=48, K=64, t=_lib.BF16,
             dt=_lib.BF16, act=4, dx=R, lddx=64, dw=S, lddw=64, db=B, work=WORK, bytes=1 << 24,
             stream=0)
    a.update(kw)
    lib = _lib.load_ffn()
    return (lib.bvml_ffn_gated_backward if gated else lib.bvml_ffn_linear_backward)(*a.values())


@pytest.mark.parametrize("gated", [False, True], ids=["linear", "gated"])
@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), _lib.FFN_ESHAPE), (dict(N=0), _lib.FFN_ESHAPE), (dict(lddy=47), _lib.FFN_ESHAPE),
    (dict(lddx=63), _lib.FFN_ESHAPE), (dict(lddw=63), _lib.FFN_ESHAPE),
    (dict(t=_lib.F32), _lib.FFN_ETYPE), (dict(t=_lib.E4M3), _lib.FFN_ETYPE),
    (dict(dt=_lib.F16), _lib.FFN_ETYPE), (dict(act=9), _lib.FFN_EPARAM),
    (dict(dy=0), _lib.FFN_ENULL), (dict(x=0), _lib.FFN_ENULL), (dict(w=0), _lib.FFN_ENULL),
    (dict(z=0), _lib.FFN_ENULL), (dict(dx=Y), _lib.FFN_EALIAS), (dict(dw=R), _lib.FFN_EALIAS),
    (dict(db=W), _lib.FFN_EALIAS), (dict(work=0), _lib.FFN_EWORK), (dict(bytes=9), _lib.FFN_EWORK),
    (dict(work=WORK + 4), _lib.FFN_EWORK), (dict(work=X), _lib.FFN_EALIAS),
    (dict(dx=0, dw=0, db=0, work=0), _lib.OK)])
def test_backward_refuses(kw, code, gated):
    assert grads(gated, **kw) == code
    if code:
        assert _lib.ffn_last_error().startswith("gated_backward: " if gated
                                                else "linear_backward: ")


def test_workspaces():
    lib = _lib.load_ffn()
    for M, N, K in ((0, 1, 1), (1, 1, 1), (63, 5, 4096), (65, 64, 64), (1000, 40, 8192)):
        assert lib.bvml_ffn_linear_workspace(M, N, K, _lib.BF16) >= 0
        assert lib.bvml_ffn_gated_workspace(M, N, K, _lib.E4M3) >= 0
        # dz at least
        assert lib.bvml_ffn_linear_backward_workspace(M, N, K) >= 2 * M * N
        assert lib.bvml_ffn_gated_backward_workspace(M, N, K) >= 4 * M * N
        assert lib.bvml_ffn_add_rms_norm_backward_workspace(M, N) >= 0
    assert lib.bvml_ffn_linear_workspace(-1, 1, 1, _lib.BF16) == -1
    assert lib.bvml_ffn_gated_backward_workspace(1, 0, 1) == -1
    assert lib.bvml_ffn_add_rms_norm_backward_workspace(1, 0) == -1


@pytest.mark.parametrize("call,message", [
    (lambda x: ffn.linear(x, x), "HIP device"), (lambda x: ffn.gated(x, x), "HIP device"),
    (lambda x: ffn.add_rms_norm(x), "HIP device"),
    (lambda x: ffn.add_rms_norm_backward(x, x, None, x), "HIP device"),
    (lambda x: ffn.linear_backward(x, x, x), "HIP device"),
])
def test_python_refuses_cpu_tensors(call, message):
    with pytest.raises(RuntimeError, match="ffn ops: .*" + message):
        call(torch.zeros(4, 4, dtype=torch.bfloat16))


def test_rows_of_views():
    t = torch.zeros(4, 6, 8)
    assert ffn._rows("op", "x", t) == (24, 8, 8)
    assert ffn._rows("op", "x", t[:, :, :5]) == (24, 5, 8)
    assert ffn._rows("op", "x", t[0, 0]) == (1, 8, 8)
    assert ffn._rows("op", "x", t[:, 2]) == (4, 8, 48)
    assert ffn._rows("op", "x", t[:, :1]) == (4, 8, 48)
    assert ffn._rows("op", "x", t[:0])[0] == 0
    for bad in (t[:, :3], t.transpose(0, 1), t.transpose(1, 2), t[..., ::2]):
        with pytest.raises(RuntimeError, match="ffn ops: op: x's"):
            ffn._rows("op", "x", bad)


def test_plan_reaches_every_kernel():
    """The sizes of tests/test_gpu_ffn.py name every tile, copy and split of
    the forward products and of both gradients together."""
    from tests import test_gpu_ffn as t
    seen = set()
    for M, N, K in t.FORWARD:
        for gated in (False, True):
            aligned = K % 8 == 0
            tile, deep, _, splits = _lib.ffn_plan(M, N * (1 + gated), K, _lib.BF16, 0, gated, aligned)
            seen.add((tile, deep, aligned, splits > 1))
    want = {(0, False, a, False) for a in (True, False)}
    want |= {(256, False, True, False), (128, False, True, False), (128, True, True, False),
             (64, False, True, False), (64, False, True, True), (64, True, True, False),
             (64, True, True, True), (128, False, False, False), (128, False, False, True),
             (64, True, False, False), (64, True, False, True)}
    assert want <= seen, want - seen
    seen = set()
    for M, N, K in t.GRADIENTS:
        for R in (N, 2 * N):
            tile, deep, whole, splits = _lib.ffn_plan(M, R, K, _lib.BF16, 3)
            if K % 8 == 0:
                seen.add((tile, deep, splits > 1))
    want = {(256, False, False), (256, False, True), (128, False, False), (128, False, True),
            (128, True, False), (64, False, False), (64, False, True), (64, True, False),
            (64, True, True)}
    assert want <= seen, want - seen


def test_usual_call_declines_the_rest():
    """The C form of the usual call returns None, with no error left set and no
    reference kept, for whatever is not a tensor of its own on a HIP device."""
    call = ffn._call()
    x = torch.zeros(4, 4, dtype=torch.bfloat16)
    odd = (x, x.float(), x[:, ::2], x.to(torch.float8_e4m3fn), torch.zeros(0), torch.zeros(()),
           torch.zeros([1] * 9), None, 3, "x", object())
    own = [o for o in odd if o is not None and not isinstance(o, (int, str))]  # shared by others
    before = [sys.getrefcount(o) for o in own]
    for a in odd:
        for b in odd:
            assert call.product(a, b, None, "none", None, False, None) is None
            assert call.product(x, a, b, "silu", None, True, torch.bfloat16) is None
            assert call.norm(a, b, x, 1e-6, None) is None
            assert call.norm(x, x, a, b, torch.float32) is None
    assert call.product(x, x, None, [], None, False, None) is None
    del a, b
    assert [sys.getrefcount(o) for o in own] == before
    with pytest.raises(TypeError):
        call.product(x)
    with pytest.raises(TypeError):
        call.norm(x)
