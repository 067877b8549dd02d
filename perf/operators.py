"""The dense operators of the hybrid block as measured cases: layer norm, and the linear map with its epilogue.

``norm``: ``y = (x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, and its backward pass.
``linear``: ``y = act(x @ weight.T + bias) + residual``, and its backward pass.

With ``own`` false, ``run`` computes them from elementary torch operations in float32; with ``own`` true it calls
``qkan_b200.functional``. A "train" case is the forward and the backward pass together, a "forward" case what
inference runs.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# relu is left out of the draws: its derivative jumps at 0, and two orders of the same sum fall on either side of it
ACTS = ("none", "silu", "gelu", "gelu_tanh", "tanh", "sigmoid")

#: the most that a drawn case may cost: the work of the largest listed one
MOST_FLOPS = 6 * 8192 * 4096 * 4096
MOST_NORM = 16384 * 4096


def _norm(name, mode, dtype, rows, dim, params="same", affine=True):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype, "rows": rows, "dim": dim, "params": params,
            "affine": affine}


def _linear(name, mode, dtype, rows, fan_in, fan_out, act="none", bias=True, residual=False):
    return {"name": name, "op": "linear", "mode": mode, "dtype": dtype, "rows": rows, "in": fan_in, "out": fan_out,
            "act": act, "bias": bias, "residual": residual}


def listed():
    return [
        # one token in front of the hybrid block (768 features): nothing but latency
        _norm("norm_token", "forward", "bf16", 1, 768),
        # a short batch of odd width: no row starts on a 16-byte boundary
        _norm("norm_ragged", "train", "fp32", 333, 1037),
        # the hybrid block's own shape, bfloat16 activations over float32 parameters
        _norm("norm_block", "train", "bf16", 8192, 768, params="fp32"),
        # wide float32 rows, far larger than the L2 cache
        _norm("norm_wide", "train", "fp32", 16384, 4096),
        # one token through a square projection: the weight matrix is read once
        _linear("linear_token", "forward", "bf16", 1, 4096, 4096, act="silu"),
        # 48 sequences decoded together, projection back into the residual stream
        _linear("linear_decode", "forward", "bf16", 48, 2048, 2048, residual=True),
        # the hybrid block's narrow projection into the QKAN layer
        _linear("linear_down", "train", "bf16", 8192, 768, 10),
        # and back, with the block's input added
        _linear("linear_up", "train", "bf16", 8192, 10, 768, residual=True),
        # first half of a Linear-SiLU-Linear head on image rows
        _linear("linear_head", "train", "fp32", 1024, 784, 128, act="silu"),
        # a plain float32 projection over a long batch
        _linear("linear_long", "train", "fp32", 65536, 256, 256),
        # nothing divides a tile, no row is aligned
        _linear("linear_odd", "train", "bf16", 1501, 517, 333, act="gelu"),
        # a large training step: bound by the tensor cores
        _linear("linear_large", "train", "bf16", 8192, 4096, 4096, act="silu"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """Log-uniform; two in three on a multiple of 8, the others wherever they fall."""
    n = _spread(rng, low, high)
    return n if rng.random() < 0.34 else max(8, n // 8 * 8)


def draw(rng):
    dtype = rng.choice(("bf16", "fp32"))
    mode = rng.choice(("forward", "train", "train"))
    if rng.random() < 0.4:
        dim = _size(rng, 16, 8192)
        rows = _spread(rng, 1, min(65536, max(1, MOST_NORM // dim)))
        return {"op": "norm", "mode": mode, "dtype": dtype, "rows": rows, "dim": dim,
                "params": rng.choice(("same", "fp32")), "affine": rng.random() < 0.8}
    fan_in, fan_out = _size(rng, 8, 4096), _size(rng, 8, 4096)
    # float32 rates are a fraction of bfloat16 ones: a quarter of the work at most
    most = MOST_FLOPS / (6 if dtype == "bf16" else 24) / fan_in / fan_out
    rows = _spread(rng, 1, max(1, min(65536, int(most))))
    return {"op": "linear", "mode": mode, "dtype": dtype, "rows": rows, "in": fan_in, "out": fan_out,
            "act": rng.choice(ACTS), "bias": rng.random() < 0.8, "residual": rng.random() < 0.5}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]
    s = dict(case)
    M = case["rows"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] == "norm":
        D = case["dim"]
        pt = dt if case["params"] == "same" else torch.float32
        # rows of a residual stream: each has its own scale and offset
        s["x"] = (normal(M, D) * (0.5 + normal(M, 1).abs()) + 0.5 * normal(M, 1)).to(dt)
        s["weight"] = (1 + 0.2 * normal(D)).to(pt) if case["affine"] else None
        s["bias"] = (0.2 * normal(D)).to(pt) if case["affine"] else None
        s["gy"] = normal(M, D).to(dt) if case["mode"] == "train" else None
        return s
    K, N = case["in"], case["out"]
    s["x"] = normal(M, K).to(dt)
    s["weight"] = (normal(N, K) / math.sqrt(K)).to(dt)
    s["bias"] = (0.1 * normal(N)).to(dt) if case["bias"] else None
    s["residual"] = normal(M, N).to(dt) if case["residual"] else None
    s["gy"] = normal(M, N).to(dt) if case["mode"] == "train" else None
    return s


# ------------------------------------------------------------------ plain forms
def _plain_norm(s):
    dt = s["x"].dtype
    x = s["x"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xhat = xc * rstd
    w = s["weight"].float() if s["affine"] else None
    y = xhat * w + s["bias"].float() if s["affine"] else xhat
    out = {"y": y.to(dt)}
    if s["mode"] == "train":
        gy = s["gy"].float()
        gw = gy * w if s["affine"] else gy
        dx = (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True)) * rstd
        out["grad_x"] = dx.to(dt)
        if s["affine"]:
            out["grad_weight"] = (gy * xhat).sum(0).to(s["weight"].dtype)
            out["grad_bias"] = gy.sum(0).to(s["weight"].dtype)
    return out


def _plain_act(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, None
    if act == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if act == "gelu":
        half = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * half, half + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    sg = 1 / (1 + torch.exp(-z))
    if act == "sigmoid":
        return sg, sg * (1 - sg)
    return z * sg, sg * (1 + z * (1 - sg))


def _plain_linear(s):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, slope = _plain_act(z, s["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dt)}
    if s["mode"] == "train":
        gz = s["gy"].float() if slope is None else s["gy"].float() * slope
        out["grad_x"] = (gz @ w).to(dt)
        out["grad_weight"] = (gz.t() @ x).to(dt)
        if s["bias"] is not None:
            out["grad_bias"] = gz.sum(0).to(dt)
    return out


# ------------------------------------------------------------------ the framework's calls
def _own_norm(s):
    from qkan_b200 import functional as F

    if s["mode"] != "train":
        return {"y": F.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)}
    y, stats = F.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=EPS)
    want = ("x", "weight", "bias") if s["affine"] else ("x",)
    g = F.layer_norm_backward(s["x"], s["weight"], stats, s["gy"], want=want)
    return {"y": y, **{"grad_" + k: v for k, v in g.items()}}


def _own_linear(s):
    from qkan_b200 import functional as F

    if s["mode"] != "train":
        return {"y": F.fused_linear(s["x"], s["weight"], s["bias"], activation=s["act"], residual=s["residual"])}
    y, tape = F.linear_forward(s["x"], s["weight"], s["bias"], activation=s["act"], residual=s["residual"],
                               return_tape=True)
    want = ("x", "weight", "bias") if s["bias"] is not None else ("x", "weight")
    g = F.linear_backward(s["x"], s["weight"], s["gy"], tape=tape, activation=s["act"], want=want)
    return {"y": y, **{"grad_" + k: v for k, v in g.items()}}


def run(state):
    if state["op"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_linear(state) if own else _plain_linear(state)


def work(case):
    M, el = case["rows"], 2 if case["dtype"] == "bf16" else 4
    train = case["mode"] == "train"
    if case["op"] == "norm":
        D = case["dim"]
        pel = el if case["params"] == "same" else 4
        vectors = (4 if train else 2) * D * pel if case["affine"] else 0
        return {"bytes": (5 if train else 2) * M * D * el + vectors, "flops": (20 if train else 8) * M * D}
    K, N = case["in"], case["out"]
    n = M * K + N * K + M * N + (N if case["bias"] else 0) + (M * N if case["residual"] else 0)
    if train:  # grad_y read; grad_x, grad_weight and grad_bias written; x and weight count once in the whole pass
        n += M * N + M * K + N * K + (N if case["bias"] else 0)
    return {"bytes": n * el, "flops": (6 if train else 2) * M * N * K}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """The operators as torch defines them, in float64, their gradients by differentiation."""
    s = prepare(case, seed)
    nn = torch.nn.functional
    leaf = {k: s[k].double().requires_grad_(case["mode"] == "train") for k in ("x", "weight", "bias")
            if s.get(k) is not None}
    if case["op"] == "norm":
        y = nn.layer_norm(leaf["x"], (case["dim"],), leaf.get("weight"), leaf.get("bias"), EPS)
    else:
        y = nn.linear(leaf["x"], leaf["weight"], leaf.get("bias"))
        act = case["act"]
        if act == "gelu_tanh":
            y = nn.gelu(y, approximate="tanh")
        elif act != "none":
            y = {"silu": nn.silu, "gelu": nn.gelu, "tanh": torch.tanh, "sigmoid": torch.sigmoid}[act](y)
        if case["residual"]:
            y = y + s["residual"].double()
    out = {"y": y.detach()}
    if case["mode"] == "train":
        grads = torch.autograd.grad(y, list(leaf.values()), s["gy"].double())
        out.update({"grad_" + k: v for k, v in zip(leaf, grads)})
    return out
