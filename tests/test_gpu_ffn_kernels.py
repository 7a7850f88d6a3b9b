"""Every kernel of the feed-forward products and of their gradients, each plan of
whole and split tiles, on its own size.  SIZES holds for every (operator, type,
copy, tile, LDS slots, state of the sums) that the launch plan can name the
smallest size found that takes it, ragged in every direction;
tests/test_ffn_plans.py checks that it leaves none out."""
from __future__ import annotations

import pytest
import torch

from brovisionml_amd import ffn
from tests import ffn_oracle as orc
from tests.test_gpu_ffn import BF, FP, HF, gen, quantised, say, within

pytestmark = pytest.mark.gpu

# (M, N, K): rows, outputs (gated: of each half), inputs
SIZES = {
    "linear": [(1, 1, 1), (2, 1, 1), (3, 1, 1), (5, 1, 1), (1, 1, 8), (2, 1, 8), (17, 1, 1),
        (3, 1, 8), (33, 1, 1), (5, 1, 8), (17, 1, 8), (33, 1, 8), (3, 4136, 1), (5, 1, 4504),
        (34, 1, 868), (3, 4100, 8), (17087, 65, 1), (16495, 65, 8), (16603, 129, 8),
        (16491, 387, 8), (471, 1399, 2458), (548, 589, 5544), (1482, 1355, 1120),
        (1350, 747, 4552), (10900, 140, 3772), (1579, 5021, 742), (2500, 1540, 2048),
        (1620, 2527, 1936), (6864, 2319, 736), (1156, 1748, 8048), (10909, 184, 9160),
        (4785, 3561, 1288), (1159, 1693, 16384)],
    "gated": [(1, 1, 1), (2, 1, 1), (3, 1, 1), (5, 1, 1), (1, 1, 8), (2, 1, 8), (17, 1, 1),
        (3, 1, 8), (33, 1, 1), (5, 1, 8), (17, 1, 8), (33, 1, 8), (5, 1, 3264), (36, 1, 724),
        (16542, 65, 8), (16387, 194, 8), (1420, 714, 1104), (607, 531, 4984), (2588, 1553, 771),
        (1188, 1677, 1856), (1602, 1258, 2024), (2274, 3599, 736), (1378, 721, 7392),
        (2728, 3047, 1248), (897, 1357, 13384)],
    "linear e4m3": [(1, 1, 1), (2, 1, 1), (3, 1, 1), (5, 1, 1), (1, 1, 16), (18, 1, 1),
        (2, 1, 16), (34, 1, 1), (3, 1, 16), (5, 1, 16), (17, 1, 16), (33, 1, 16), (3, 4162, 1),
        (5, 1, 8976), (34, 2, 1737), (3, 4097, 16), (16497, 65, 2), (16903, 65, 16),
        (16936, 129, 16), (16499, 392, 16), (456, 732, 10768), (869, 855, 5497),
        (1540, 1452, 2080), (1052, 1013, 9552), (10883, 154, 6443), (1830, 4461, 1571),
        (1164, 3449, 4016), (2560, 1602, 4224), (2890, 5744, 1808), (1719, 1153, 15920),
        (6598, 2549, 2416)],
    "gated e4m3": [(1, 1, 1), (2, 1, 1), (3, 1, 1), (5, 1, 1), (1, 1, 16), (17, 1, 1), (2, 1, 16),
        (33, 1, 1), (3, 1, 16), (5, 1, 16), (17, 1, 16), (33, 1, 16), (5, 1, 6416), (33, 1, 1432),
        (16416, 65, 16), (16492, 193, 16), (1094, 1029, 2144), (479, 689, 10224),
        (3884, 1051, 1435), (1302, 1575, 4144), (1632, 1246, 4256), (1217, 780, 15104),
        (2548, 3305, 2032), (3741, 2185, 2320)],
    "input": [(1, 1, 1), (1, 1, 8), (1, 711, 1), (1, 1858, 8), (65, 1, 16416), (66, 1, 16477),
        (16582, 1, 136), (16503, 3, 392), (851, 2217, 853), (661, 5036, 504), (1639, 966, 1224),
        (1350, 4132, 736), (2139, 763, 3873), (1688, 1709, 2424), (2544, 1893, 1640),
        (5095, 765, 3272), (6578, 7217, 288), (2255, 852, 7184), (1718, 6979, 1248),
        (2327, 8014, 2184)],
    "weight": [(1, 1, 1), (1, 1, 8), (705, 1, 1), (1731, 1, 8), (1, 65, 16920), (1, 193, 16632),
        (3, 68, 16452), (1, 515, 14552), (1957, 969, 654), (4738, 693, 512), (871, 1753, 1184),
        (3896, 860, 1160), (718, 2314, 3372), (1593, 3639, 1096), (1782, 2789, 1512),
        (5720, 6537, 320), (760, 2985, 5512), (786, 5713, 2824), (6144, 1816, 1152),
        (8540, 2692, 760)],
    "both": [(1, 1, 8), (1, 65, 8), (1, 961, 8), (961, 1, 8), (1, 1, 16448), (1, 65, 11120),
        (15118, 1, 72), (970, 257, 8), (260, 1092, 8), (2, 7390, 200), (1224, 2135, 8),
        (1286, 2183, 8), (65, 76, 16608), (65, 131, 13136), (214, 2020, 712), (323, 714, 1808),
        (1837, 344, 672), (684, 419, 1800), (197, 205, 16888), (2640, 594, 456), (2485, 738, 408),
        (723, 3208, 328), (2826, 3875, 72), (3567, 3083, 72), (588, 2238, 624), (259, 323, 12056),
        (454, 3212, 832), (589, 3723, 664), (3343, 636, 800), (4988, 4406, 80), (4008, 5498, 80),
        (3978, 723, 672), (1485, 1865, 1160), (1923, 1622, 1152), (1956, 1697, 1120),
        (1717, 1953, 1152), (9172, 7385, 80), (706, 736, 10936), (8959, 6100, 104),
        (970, 6262, 936), (6595, 3326, 264), (6811, 1155, 816), (1531, 1774, 2560),
        (7575, 1416, 656), (981, 7917, 944), (2033, 2102, 1984), (1190, 1497, 6144),
        (7056, 4941, 456), (7233, 5193, 496)],
}
HALVES = pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])


def sizes(name):
    return pytest.mark.parametrize("M,N,K", SIZES[name])


@HALVES
@sizes("linear")
def test_linear(cuda, M, N, K, dtype):
    say(f"linear {M}x{K}x{N} {dtype}")
    rnd = gen(M + N + K)
    x, w = rnd(M, K).to(dtype), rnd(N, K, std=K ** -0.5).to(dtype)
    b, r = rnd(N, std=0.3).to(dtype), rnd(M, N).to(dtype)
    got = ffn.linear(x, w, b, "gelu", r, save=True)
    within("y", got.y, *orc.linear(x, w, b, "gelu", r, dtype))
    z, ez = orc.pre(x, w, b)
    within("z", got.z, z, ez + orc.stored(z.abs() + ez, dtype))


@HALVES
@sizes("gated")
def test_gated(cuda, M, N, K, dtype):
    say(f"gated {M}x{K}x{N} {dtype}")
    rnd = gen(M + N + K)
    x, w = rnd(M, K).to(dtype), rnd(2 * N, K, std=K ** -0.5).to(dtype)
    b = rnd(2 * N, std=0.3)
    got = ffn.gated(x, w, b, "silu", save=True)
    within("h", got.y, *orc.gated(x, w, b, "silu", dtype))
    z, ez = orc.pre(x, w, b)
    within("z", got.z, z, ez + orc.stored(z.abs() + ez, dtype))


@sizes("linear e4m3")
def test_linear_e4m3(cuda, M, N, K):
    say(f"linear e4m3 {M}x{K}x{N}")
    rnd = gen(M + N + K)
    (x, xs), (w, ws) = quantised(rnd(M, K)), quantised(rnd(N, K, std=K ** -0.5))
    out = (BF, HF, FP)[(M + N + K) % 3]
    b, r = rnd(N, std=0.2).to(out), rnd(M, N).to(out)
    got = ffn.linear(x, w, b, "gelu", r, x_scale=xs, w_scale=ws, dtype=out).y
    within("y", got, *orc.linear(x, w, b, "gelu", r, out, xs, ws))


@sizes("gated e4m3")
def test_gated_e4m3(cuda, M, N, K):
    say(f"gated e4m3 {M}x{K}x{N}")
    rnd = gen(M + N + K)
    (x, xs), (w, ws) = quantised(rnd(M, K)), quantised(rnd(2 * N, K, std=K ** -0.5))
    out = (BF, HF, FP)[(M + N + K) % 3]
    b = rnd(2 * N, std=0.2).to(out)
    got = ffn.gated(x, w, b, "silu", x_scale=xs, w_scale=ws, dtype=out).y
    within("h", got, *orc.gated(x, w, b, "silu", out, xs, ws))


def gradients(M, N, K, dtype):
    """dy, x, w, z with an activation, so that dz is the kernels' own array, whose
    rows begin on 16 bytes."""
    rnd = gen(M + N + K)
    return (rnd(M, N, std=0.3).to(dtype), rnd(M, K).to(dtype), rnd(N, K, std=K ** -0.5).to(dtype),
            rnd(M, N).to(dtype))


@HALVES
@sizes("input")
def test_input_gradient(cuda, M, N, K, dtype):
    say(f"dx {M}x{K}x{N} {dtype}")
    dy, x, w, z = gradients(M, N, K, dtype)
    dx, dw, db = ffn.linear_backward(dy, x, w, z, "silu", need_w=False, need_bias=False)
    assert dw is None and db is None
    within("dx", dx, *orc.grads(dy, x, w, z, "silu", False, dtype)[0])


@HALVES
@sizes("weight")
def test_weight_gradient(cuda, M, N, K, dtype):
    say(f"dw {M}x{K}x{N} {dtype}")
    dy, x, w, z = gradients(M, N, K, dtype)
    dx, dw, db = ffn.linear_backward(dy, x, w, z, "silu", need_x=False)
    assert dx is None
    want = orc.grads(dy, x, w, z, "silu", False, dtype)
    within("dw", dw, *want[1])
    within("db", db, *want[2])


@HALVES
@sizes("both")
def test_both_gradients(cuda, M, N, K, dtype):
    say(f"gradients {M}x{K}x{N} {dtype}")
    dy, x, w, z = gradients(M, N, K, dtype)
    got = ffn.linear_backward(dy, x, w, z, "silu")
    for name, g, want in zip(("dx", "dw", "db"), got, orc.grads(dy, x, w, z, "silu", False, dtype)):
        within(name, g, *want)
