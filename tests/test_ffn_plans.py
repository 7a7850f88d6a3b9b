"""The launch plan without a GPU: tests/test_gpu_ffn_kernels.py's sizes name every
kernel and every plan of whole and split tiles that thousands of other sizes name."""
from __future__ import annotations

import math
import random

import pytest

from brovisionml_amd import _lib
from tests.test_gpu_ffn_kernels import SIZES

# rows of a tile and its LDS slots; each product's sums: a workgroup a tile
# ("one"), every tile split, or whole tiles and split ones together ("both")
TILES = [(256, False), (128, False), (128, True), (64, False), (64, True)]


def state(whole, splits):
    return "one" if splits == 1 else "split" if whole == 0 else "both"


def kernel(name, M, N, K):
    """What a call of operator `name` of these sizes launches."""
    e4m3, gated = name.endswith("e4m3"), name.startswith("gated")
    aligned = K % (16 if e4m3 else 8) == 0
    if name == "input":
        plan = _lib.ffn_plan(M, K, N, _lib.BF16, 1, False, aligned)
    elif name == "weight":
        plan = _lib.ffn_plan(N, K, M, _lib.BF16, 2, False, aligned)
    elif name == "both":
        plan = _lib.ffn_plan(M, N, K, _lib.BF16, 3)
    else:
        plan = _lib.ffn_plan(M, N * (1 + gated), K, _lib.E4M3 if e4m3 else _lib.BF16, 0, gated,
                             aligned)
    tile, slots, whole, splits = plan
    if tile:
        return (tile, slots), aligned, state(whole, splits)
    # few rows: one, two, up to four (a wave of one or two columns), 16, 32
    rows = next(m for m in (1, 2, 4, 16, 32) if M <= m)
    return rows, aligned, rows == 4 and N >= 4096 and not gated


def covered(name):
    return {kernel(name, *size) for size in SIZES[name]}


@pytest.mark.parametrize("name", SIZES)
def test_sizes_reach_what_the_plan_names(name):
    rng, seen = random.Random(name), covered(name)
    e4m3, missing = name.endswith("e4m3"), {}

    def size(most):
        return round(math.exp(rng.uniform(0, math.log(most))))

    for _ in range(30000):
        M, N, K = size(20000), size(9000), size(18000)
        piece = 16 if e4m3 else 8
        if name == "both" or rng.random() < 0.7:
            K = max(piece, K // piece * piece)
        if M * N * K > 6e10:  # as large as a test should be
            continue
        k = kernel(name, M, N, K)
        if k not in seen:
            missing.setdefault(k, (M, N, K))
    assert not missing


@pytest.mark.parametrize("name", SIZES)
def test_every_tile_is_among_them(name):
    """By hand, so that a change of the plan that no longer names a kernel is
    seen as well."""
    got = {k[:2] for k in covered(name) if isinstance(k[0], tuple)}
    want = {(tile, True) for tile in TILES}
    if name.startswith("gated"):
        want.remove(((64, True), True))
    if name != "both":  # through registers
        want |= {((128, False), False)}
        if not name.startswith("gated"):
            want |= {((64, True), False)}
    assert got == want
    sums = {(k[0], k[2]) for k in covered(name) if isinstance(k[0], tuple) and k[1]}
    for tile in ((256, False), (128, False), (128, True)):
        for s in ("one", "both"):
            assert (tile, s) in sums, (tile, s)
