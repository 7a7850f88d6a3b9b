"""The feed-forward half of a pre-norm transformer block, as measurable cases.

Three operators, each forward and backward, as a program that runs a
transformer encoder beside the refiner calls them on tensors on the GPU:

  norm     s = x + r, y = s / sqrt(mean(s^2) + eps) * w; y in 16 bits or in
           e4m3 with one scale a row, s as the new residual stream
  linear   y = act(x W^T + b) + r, x and W in 16 bits or in e4m3 with a scale
           for each row of x and of W
  gated    h = act(x Wg^T + bg) * (x Wu^T + bu), W = [Wg; Wu] stacked

Token counts are those of the repository's grids (60x80 and 13x19 patches
and five more tokens, 256x256 rows), a single token, small batches of single
tokens and generic long batches; widths are generic encoder widths (1024,
1280, four times those, 8/3 of 1024, a 1000-way head).
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
TINY = 2.0 ** -126
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
          "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # the norm: one token while serving; an encoder's 60x80 patches with
        # a 32-bit residual stream, quantised for 8-bit products; the
        # gradient of a long batch
        {"name": "norm 1x1280 bf16", "op": "norm", "T": 1, "K": 1280, "x": "bf16", "y": "bf16"},
        {"name": "norm 4805x1280 f32 to e4m3", "op": "norm", "T": 4805, "K": 1280, "x": "f32",
         "y": "e4m3"},
        {"name": "norm backward 65541x1024", "op": "norm_backward", "T": 65541, "K": 1024,
         "x": "bf16", "y": "bf16"},
        # the product: the down projection of one token; a 1000-way head on a
        # 13x19 grid; the down projection of 60x80 patches; the up projection
        # in 8 bits; the gradient of a projection with its activation
        {"name": "linear 1x5120x1280 bf16", "op": "linear", "T": 1, "K": 5120, "N": 1280,
         "x": "bf16", "y": "bf16", "act": "none", "residual": True},
        {"name": "linear 252x1024x1000 f16", "op": "linear", "T": 252, "K": 1024, "N": 1000,
         "x": "f16", "y": "f16", "act": "gelu", "residual": False},
        {"name": "linear 4805x5120x1280 bf16", "op": "linear", "T": 4805, "K": 5120, "N": 1280,
         "x": "bf16", "y": "bf16", "act": "none", "residual": True},
        {"name": "linear 4805x1280x5120 e4m3", "op": "linear", "T": 4805, "K": 1280, "N": 5120,
         "x": "e4m3", "y": "bf16", "act": "gelu_tanh", "residual": False},
        {"name": "linear backward 4805x1280", "op": "linear_backward", "T": 4805, "K": 1280,
         "N": 5120, "x": "bf16", "y": "bf16", "act": "gelu"},
        # the gated block: a batch of four single tokens; 60x80 patches, with
        # what the backward pass needs; its gradient, of a ragged width and
        # of a long batch
        {"name": "gated 4x1280x5120 bf16", "op": "gated", "T": 4, "K": 1280, "N": 5120,
         "x": "bf16", "y": "bf16", "act": "silu", "save": False},
        {"name": "gated 4805x1280x5120 bf16", "op": "gated", "T": 4805, "K": 1280, "N": 5120,
         "x": "bf16", "y": "bf16", "act": "silu", "save": True},
        {"name": "gated backward 1205x1024x2730", "op": "gated_backward", "T": 1205, "K": 1024,
         "N": 2730, "x": "f16", "y": "f16", "act": "silu"},
        {"name": "gated backward 16389x1024", "op": "gated_backward", "T": 16389, "K": 1024,
         "N": 4096, "x": "bf16", "y": "bf16", "act": "gelu_tanh"},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of its range, odd ones among them."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 8 if n == 3072 else n


def _width(rng, lo, hi):
    """Mostly a whole number of 16-byte pieces, now and then any number."""
    n = _size(rng, lo, hi)
    if rng.random() < 0.85:
        n = max(8, n // 8 * 8)
    return n + 8 if n == 3072 else n


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "linear", "linear", "linear_backward", "gated",
                     "gated", "gated_backward"])
    kind = rng.choice(["bf16", "bf16", "f16"])
    if op.startswith("norm"):
        K = _width(rng, 64, 8192)
        x = rng.choice([kind, kind, "f32"])
        T = _size(rng, 1, max(2, 65541 * 1024 // (K * (2 if x == "f32" else 1))))
        y = kind
        if op == "norm" and rng.random() < 0.4:
            y = "e4m3"
        return {"op": op, "T": T, "K": K, "x": x, "y": y if y == "e4m3" or x == "f32" else x}
    K, N = _width(rng, 128, 5120), _width(rng, 128, 5120)
    # at most the work of the largest listed case
    most = 4 * 16389 * 1024 * 8192
    each = K * N * 2 * (2 if op.startswith("gated") else 1) * (2 if "backward" in op else 1)
    T = _size(rng, 1, max(2, min(16389, most // each)))
    act = rng.choice(["silu", "gelu", "gelu_tanh"]) if op.startswith("gated") \
        else rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    case = {"op": op, "T": T, "K": K, "N": N, "x": kind, "y": kind, "act": act}
    if not op.endswith("backward") and rng.random() < 0.3:
        # 16 values of 8 bits make a 16-byte piece
        case.update(x="e4m3", K=max(16, K // 16 * 16))
        if case["K"] == 3072:
            case["K"] += 16
    if op == "linear":
        case["residual"] = rng.random() < 0.5
    if op == "gated":
        case["save"] = case["x"] != "e4m3" and rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _quantised(v):
    """Rows of v as e4m3 and one scale a row."""
    scale = (v.abs().amax(-1) / E4M3_MAX).clamp(min=TINY)
    return (v / scale[:, None]).to(torch.float8_e4m3fn), scale


def _inputs(case, seed):
    """What the program has before the call, by name."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    op, T, K, x_type, y_type = (case[k] for k in ("op", "T", "K", "x", "y"))
    xt = DTYPES[x_type]
    if op.startswith("norm"):
        # a residual stream: some channels are many times larger than others
        channel = torch.exp(randn(K, std=0.8))
        w = (1.0 + randn(K, std=0.2)).to(torch.float32 if x_type == "f32" else xt)
        x = (randn(T, K) * channel).to(xt)
        if op == "norm":
            return {"x": x, "residual": (randn(T, K) * channel).to(xt), "w": w}
        s = x.float()
        return {"dy": randn(T, K, std=0.05).to(DTYPES[y_type]), "s": x, "w": w,
                "rstd": torch.rsqrt((s * s).mean(-1) + EPS),
                "dstream": randn(T, K, std=0.05).to(xt)}
    N = case["N"]
    rows = 2 * N if op.startswith("gated") else N
    x, w = randn(T, K), randn(rows, K, std=K ** -0.5)
    if x_type == "e4m3":
        (x, xs), (w, ws) = _quantised(x), _quantised(w)
        return {"x": x, "xs": xs, "w": w, "ws": ws,
                "b": randn(rows, std=0.1).to(DTYPES[y_type]),
                "residual": randn(T, N).to(DTYPES[y_type]) if case.get("residual") else None}
    x, w = x.to(xt), w.to(xt)
    if op.endswith("backward"):
        # the pre-activations that the forward pass saved
        z = (x.float() @ w.float().t() + randn(rows, std=0.1)).to(xt)
        return {"dy": randn(T, N, std=0.05).to(xt), "x": x, "w": w, "z": z}
    return {"x": x, "w": w, "b": randn(rows, std=0.1).to(xt),
            "residual": randn(T, N).to(xt) if case.get("residual") else None}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from brovisionml_amd import ffn
    case = state["case"]
    op, y_type = case["op"], DTYPES[case["y"]]
    if op == "norm":
        out = ffn.add_rms_norm(state["x"], state["residual"], state["w"], EPS, dtype=y_type)
        return [out.y, out.stream] + ([out.scale] if case["y"] == "e4m3" else [])
    if op == "norm_backward":
        return list(ffn.add_rms_norm_backward(state["dy"], state["s"], state["w"], state["rstd"],
                                              state["dstream"]))
    if op == "linear_backward":
        return list(ffn.linear_backward(state["dy"], state["x"], state["w"], state["z"],
                                        case["act"]))
    if op == "gated_backward":
        return list(ffn.gated_backward(state["dy"], state["x"], state["w"], state["z"],
                                       case["act"]))
    scales = {"x_scale": state["xs"], "w_scale": state["ws"], "dtype": y_type} \
        if case["x"] == "e4m3" else {}
    if op == "linear":
        return [ffn.linear(state["x"], state["w"], state["b"], case["act"], state["residual"],
                           **scales).y]
    out = ffn.gated(state["x"], state["w"], state["b"], case["act"], save=case["save"], **scales)
    return [out.y] + ([out.z] if case["save"] else [])


SQRT_HALF = math.sqrt(0.5)
TANH_A, TANH_B = math.sqrt(2.0 / math.pi), 0.044715


def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * SQRT_HALF))
    return 0.5 * z * (1 + torch.tanh(TANH_A * (z + TANH_B * z * z * z)))


def _act_slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * SQRT_HALF)) \
            + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    t = torch.tanh(TANH_A * (z + TANH_B * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * TANH_A * (1 + 3 * TANH_B * z * z)


def _plain(state):
    case = state["case"]
    op, y_type = case["op"], DTYPES[case["y"]]
    if op == "norm":
        s = state["x"].float() + state["residual"].float()
        y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS) * state["w"].float()
        if case["y"] == "e4m3":
            q, scale = _quantised(y)
            return [q, s.to(state["x"].dtype), scale]
        return [y.to(y_type), s.to(state["x"].dtype)]
    if op == "norm_backward":
        s, dy, rstd = state["s"].float(), state["dy"].float(), state["rstd"][:, None]
        n = s * rstd
        a = dy * state["w"].float()
        ds = rstd * (a - n * (a * n).mean(-1, keepdim=True)) + state["dstream"].float()
        return [ds.to(state["s"].dtype), (dy * n).sum(0).to(state["w"].dtype)]
    x, w = state["x"].float(), state["w"].float()
    if op.endswith("backward"):
        dy, z, kind = state["dy"].float(), state["z"].float(), state["x"].dtype
        if op == "linear_backward":
            dz = dy * _act_slope(case["act"], z)
        else:
            gate, up = z.chunk(2, -1)
            dz = torch.cat([dy * up * _act_slope(case["act"], gate),
                            dy * _act(case["act"], gate)], -1)
        return [(dz @ w).to(kind), (dz.t() @ x).to(kind), dz.sum(0).to(kind)]
    z = x @ w.t()
    if case["x"] == "e4m3":
        z = z * state["xs"][:, None] * state["ws"]
    z = z + state["b"].float()
    if op == "linear":
        y = _act(case["act"], z)
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return [y.to(y_type)]
    gate, up = z.chunk(2, -1)
    h = (_act(case["act"], gate) * up).to(y_type)
    return [h, z.to(y_type)] if case["save"] else [h]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


def work(case):
    op, T, K, xb, yb = case["op"], case["T"], case["K"], BYTES[case["x"]], BYTES[case["y"]]
    if op == "norm":
        # x, r in; y, s out; the row scales; the weight
        return {"bytes": T * K * (3 * xb + yb) + (4 * T if yb == 1 else 0) + K * xb,
                "flops": 6 * T * K}
    if op == "norm_backward":
        # dy, s, dstream in; ds out; rstd; the weight and its gradient
        return {"bytes": T * K * (yb + 3 * xb) + 4 * T + 2 * K * xb, "flops": 12 * T * K}
    N = case["N"]
    rows = 2 * N if op.startswith("gated") else N
    if op.endswith("backward"):
        # dy, x, w, z in; the three gradients out
        return {"bytes": xb * (T * (N + 2 * K + rows) + 2 * rows * K + rows),
                "flops": 4 * T * rows * K}
    outs = T * N * (2 if case.get("residual") else 1) + (T * rows if case.get("save") else 0)
    scales = 4 * (T + rows) if xb == 1 else 0
    return {"bytes": xb * K * (T + rows) + yb * (outs + rows) + scales,
            "flops": 2 * T * rows * K}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _phi64(z):
    return torch.special.ndtr(z)


def _f64(name, z):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0)
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return z * p, p + z * p * (1 - p)
    if name == "gelu":
        return z * _phi64(z), _phi64(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    # 0.5 (1 + tanh(a)) = sigmoid(2 a)
    inner = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    p = 1.0 / (1.0 + torch.exp(-inner))
    slope = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
    return z * p, p + z * p * (1 - p) * slope


def exact(case, seed):
    d = {k: v.double() if v is not None else None for k, v in _inputs(case, seed).items()}
    op, act = case["op"], case.get("act")
    if op == "norm":
        s = d["x"] + d["residual"]
        y = d["w"] * s / torch.sqrt(torch.mean(s * s, dim=1, keepdim=True) + EPS)
        if case["y"] != "e4m3":
            return [y, s]
        scale = torch.amax(torch.abs(y), dim=1) / E4M3_MAX
        return [y / scale[:, None], s, scale]
    if op == "norm_backward":
        a = d["dy"] * d["w"]
        dot = torch.sum(a * d["s"], dim=1, keepdim=True)
        r = d["rstd"][:, None]
        ds = r * a - d["s"] * r ** 3 * dot / case["K"] + d["dstream"]
        return [ds, torch.sum(d["dy"] * d["s"] * r, dim=0)]
    if op == "linear":
        z = torch.matmul(d["x"], d["w"].t().contiguous())
        if "xs" in d:
            z = z * torch.outer(d["xs"], d["ws"])
        y = _f64(act, z + d["b"])[0]
        return [y if d["residual"] is None else y + d["residual"]]
    if op == "gated":
        z = torch.matmul(d["x"], d["w"].t().contiguous())
        if "xs" in d:
            z = z * torch.outer(d["xs"], d["ws"])
        z = z + d["b"]
        h = _f64(act, z[:, :case["N"]])[0] * z[:, case["N"]:]
        return [h, z] if case["save"] else [h]
    if op == "linear_backward":
        dz = d["dy"] * _f64(act, d["z"])[1]
    else:
        gate, up = d["z"][:, :case["N"]], d["z"][:, case["N"]:]
        value, slope = _f64(act, gate)
        dz = torch.cat([d["dy"] * up * slope, d["dy"] * value], dim=1)
    return [torch.matmul(dz, d["w"]), torch.matmul(dz.t().contiguous(), d["x"]),
            torch.sum(dz, dim=0)]
