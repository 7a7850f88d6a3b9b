"""Refusals of the feed-forward operators beyond those of a single bad argument,
without a GPU: every call here fails its checks, or would before it could launch."""
from __future__ import annotations

import pytest

from brovisionml_amd import _lib
from tests.test_ffn_host import B, R, S, T, WORK, X, Y, Z, norm, norm_grad, product  # noqa: F401


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
