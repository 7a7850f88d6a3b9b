"""Refusals of the feed-forward operators beyond those of a single bad argument,
without a GPU: every call here fails its checks, or would before it could launch."""
from __future__ import annotations

import pytest
import torch

from brovisionml_amd import _lib, ffn
from tests.test_ffn_host import B, R, S, T, W, WORK, X, Y, Z, norm, norm_grad, product


# ---------------------------------------------------------------------------
# an output may be the one input that the header names, and no other
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kw,message", [
    (dict(ds=R), "ds overlaps s"),                       # s itself: only dstream may be ds
    (dict(ds=R, dstream=0), "ds overlaps s"),
    (dict(ds=X), "ds overlaps dy"),
    (dict(ds=S + 64), "ds overlaps dstream"),            # dstream, but not row for row
    (dict(ds=S, ldds=80), "ds overlaps dstream"),
])
def test_norm_backward_refuses_other_aliases(kw, message):
    # (the workspace is missing, so that nothing could be launched)
    assert norm_grad(work=0, **kw) == _lib.FFN_EALIAS
    assert _lib.ffn_last_error() == "add_rms_norm_backward: " + message


def test_the_named_aliases_pass_their_check():
    """Refused for the missing workspace, the check after the aliases'."""
    assert norm_grad(work=0, ds=S) == _lib.FFN_EWORK


@pytest.mark.parametrize("kw,message", [
    (dict(y=X), "y overlaps x"), (dict(stream=B), "stream overlaps weight"),
    (dict(stream=X + 2), "stream overlaps x"),
    (dict(stream=R, ldr=70), "stream overlaps residual")])
def test_norm_refuses_other_aliases(kw, message):
    assert norm(**kw) == _lib.FFN_EALIAS
    assert _lib.ffn_last_error() == "add_rms_norm: " + message


# ---------------------------------------------------------------------------
# the forward products' workspace, where their sums are split
# ---------------------------------------------------------------------------
SPLIT = dict(M=128, N=64, K=8192, ldx=8192, ldw=8192, ldy=64, ldr=64, ldz=128, it=_lib.BF16)


@pytest.mark.parametrize("gated,at,name", [(False, R, "residual")] + [
    (gated, at, name) for gated in (False, True)
    for at, name in ((X + 4096, "x"), (W, "w"), (W + 1024 * 1024 - 16, "w"), (B, "bias"),
                     (Y + 16, "y"), (Z, "z"))])
def test_forward_refuses_a_workspace_over_another_argument(gated, at, name):
    assert _lib.load_ffn().bvml_ffn_linear_workspace(128, 64, 8192, _lib.BF16) > 0
    assert _lib.load_ffn().bvml_ffn_gated_workspace(128, 64, 8192, _lib.BF16) > 0
    assert product(gated, work=at, **SPLIT) == _lib.FFN_EALIAS
    name = "h" if gated and name == "y" else name
    assert _lib.ffn_last_error().endswith(f": the workspace overlaps {name}")


@pytest.mark.parametrize("gated", [False, True], ids=["linear", "gated"])
def test_forward_refuses_a_workspace_off_16_bytes(gated):
    assert product(gated, work=WORK + 8, **SPLIT) == _lib.FFN_EWORK
    assert "16 bytes" in _lib.ffn_last_error()


@pytest.mark.parametrize("name,at", [("x_scale", S), ("w_scale", T)])
def test_forward_refuses_a_workspace_over_the_scales(name, at):
    kw = {**SPLIT, "it": _lib.E4M3, "K": 16384, "ldx": 16384, "ldw": 16384}
    assert _lib.load_ffn().bvml_ffn_linear_workspace(128, 64, 16384, _lib.E4M3) > 0
    assert product(work=at, xs=S, ws=T, z=0, **kw) == _lib.FFN_EALIAS
    assert _lib.ffn_last_error() == f"linear: the workspace overlaps {name}"


# ---------------------------------------------------------------------------
# sizes beyond the entry points' 32-bit integers
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(2 ** 32 + 5, 1), (2 ** 31, 8), (2 ** 16, 2 ** 16, 3),
                                   (4, 2 ** 31), (2 ** 31,)])
def test_sizes_beyond_32_bits_are_refused(shape):
    t = torch.empty(shape, dtype=torch.bfloat16, device="meta")
    with pytest.raises(RuntimeError, match="ffn ops: op: x has .* more than 2147483647"):
        ffn._rows("op", "x", t)


def test_the_largest_sizes_are_taken():
    t = torch.empty(2 ** 31 - 1, 1, dtype=torch.bfloat16, device="meta")
    assert ffn._rows("op", "x", t) == (2 ** 31 - 1, 1, 1)


def test_workspaces_of_the_most_rows():
    """dz is 16 bytes a row for one output, the rest the same for 256 runs of
    rows, however close the rows are to the largest int."""
    lib = _lib.load_ffn()
    below, most = 2 ** 31 - 2 ** 23 - 2 ** 16, 2 ** 31 - 512
    got = [lib.bvml_ffn_linear_backward_workspace(M, 1, 1) for M in (below, most)]
    assert got[1] - got[0] == 16 * (most - below)
    # 1,024 workgroups' partial rows
    assert lib.bvml_ffn_add_rms_norm_backward_workspace(2 ** 31 - 1, 64) == 1024 * 64 * 4


# ---------------------------------------------------------------------------
# more tiles than one launch holds (2^32 threads)
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("gated", [False, True], ids=["linear", "gated"])
@pytest.mark.parametrize("N", [4096, 1 << 20])
def test_more_tiles_than_a_launch_holds_are_refused(gated, N):
    """Arrays of up to 2^52 bytes at addresses 2^56 apart: refused before any
    launch."""
    at = [(i + 1) << 56 for i in range(4)]
    kw = dict(x=at[0], ldx=8, w=at[1], ldw=8, bias=0, residual=0, M=2 ** 31 - 512, N=N, K=8,
              y=at[2], ldy=N, z=0, work=at[3], bytes=1 << 40)
    assert product(gated, **kw) == _lib.FFN_ESIZE
    assert "more tiles than a launch holds" in _lib.ffn_last_error()


@pytest.mark.parametrize("shape", [(3, 0, 64), (0, 5, 64), (3, 0, 2, 64), (2, 3, 0, 64), (0, 64)])
def test_no_rows_in_any_dimension(shape):
    t = torch.zeros(shape)
    assert ffn._rows("op", "x", t)[:2] == (0, 64)
    wide = torch.zeros(*shape[:-1], 100)[..., :64]
    assert ffn._rows("op", "x", wide)[:2] == (0, 64)


@pytest.mark.parametrize("eps", [1e39, 1e308, float("inf")])
def test_norm_refuses_an_eps_that_fp32_does_not_hold(eps):
    # (no rows: nothing could be launched)
    assert norm(rows=0, eps=eps) == _lib.FFN_EPARAM
    assert norm(rows=0, eps=3e38) == _lib.OK
