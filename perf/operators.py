"""Cases of the 8-bit serving operators: what they compute, in plain torch and in 64 bits, and what they have to move.

* ``linear``: product of 8-bit codes with a scale per row (token) and per output channel, bias, activation
* ``norm``: residual addition, root-mean-square norm, 8-bit codes with a scale per row
* ``quantize``: floating rows to 8-bit codes with a scale per row, and back to floating point
* ``policy``: the three layers of a policy network on 8-bit codes

Codes are compared as the values they stand for (code times scale), in a 16-bit type.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # a policy's 400-wide hidden layer for one state: launch latency
        {"name": "linear 1x400x400", "op": "linear", "M": 1, "N": 400, "K": 400, "act": "relu", "bias": True, "type": "fp32"},
        # one token through a wide layer: the weights' bytes
        {"name": "linear 1x16384x4096", "op": "linear", "M": 1, "N": 16384, "K": 4096, "act": "none", "bias": False, "type": "bf16"},
        # a learner's batch through the same hidden layer
        {"name": "linear 256x400x400", "op": "linear", "M": 256, "N": 400, "K": 400, "act": "relu", "bias": True, "type": "fp32"},
        # a ragged prompt through an odd layer: nothing is a multiple of a tile
        {"name": "linear 777x1333x2001", "op": "linear", "M": 777, "N": 1333, "K": 2001, "act": "tanh", "bias": True, "type": "fp16"},
        # a long prompt through a square layer: the matrix rate
        {"name": "linear 8192x8192x8192", "op": "linear", "M": 8192, "N": 8192, "K": 8192, "act": "none", "bias": False, "type": "bf16"},
        # one token between two layers of a residual network
        {"name": "norm 1x4096", "op": "norm", "M": 1, "K": 4096, "residual": True, "type": "bf16"},
        # a prompt between two layers
        {"name": "norm 4096x4096", "op": "norm", "M": 4096, "K": 4096, "residual": True, "type": "bf16"},
        # odd rows of full precision, the first layer (nothing to add yet)
        {"name": "norm 1023x1111", "op": "norm", "M": 1023, "K": 1111, "residual": False, "type": "fp32"},
        # hidden activations of a batch of 4096 environments
        {"name": "quantize 4096x400", "op": "quantize", "M": 4096, "K": 400, "type": "fp32"},
        # a square layer's weights, per output channel
        {"name": "quantize 8192x8192", "op": "quantize", "M": 8192, "K": 8192, "type": "bf16"},
        # one state of the walker through a 400-wide policy
        {"name": "policy 1x24-400-4", "op": "policy", "M": 1, "S": 24, "H": 400, "A": 4},
        # 4096 ants through a policy too wide for one workgroup's LDS tiles
        {"name": "policy 4096x111-1024-8", "op": "policy", "M": 4096, "S": 111, "H": 1024, "A": 8},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "norm", "norm", "quantize", "policy"])
    kind = rng.choice(["fp32", "bf16", "fp16"])
    if op == "linear":
        M = rng.choice([_log(rng, 1, 16), _log(rng, 1, 8192), _log(rng, 64, 8192)])
        return {"op": op, "M": M, "N": _log(rng, 1, 8192), "K": _log(rng, 1, 8192),
                "act": rng.choice(["none", "relu", "tanh"]), "bias": rng.random() < 0.5, "type": kind}
    if op == "norm":
        K = _log(rng, 1, 16384)
        return {"op": op, "M": _log(rng, 1, min(16384, (1 << 24) // K)), "K": K, "residual": rng.random() < 0.5, "type": kind}
    if op == "quantize":
        K = _log(rng, 1, 16384)
        return {"op": op, "M": _log(rng, 1, min(16384, (1 << 25) // K)), "K": K, "type": kind}
    return {"op": op, "M": _log(rng, 1, 8192), "S": _log(rng, 3, 376), "H": _log(rng, 64, 2048), "A": _log(rng, 1, 32)}


# ---------------------------------------------------------------------------------------------------------- inputs
def _codes(values):
    """Codes and scales of ``values`` [rows, K], in rows of a multiple of 16 bytes, as a program keeps them."""
    rows, K = values.shape
    top = values.abs().amax(1).clamp_min(1e-30)
    ld = -(-K // 16) * 16
    buf = torch.zeros(rows, ld, dtype=torch.int8, device=values.device)
    buf[:, :K] = torch.round(values * (127.0 / top)[:, None]).to(torch.int8)
    return buf[:, :K], top / 127.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case)
    op = case["op"]
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["q"], s["scale"] = _codes(normal(M, K))
        s["weight"], s["weight_scale"] = _codes(normal(N, K) / math.sqrt(K))
        s["b"] = normal(N) if case["bias"] else None
    elif op == "norm":
        M, K, t = case["M"], case["K"], _TYPES[case["type"]]
        s["x"] = normal(M, K).to(t)
        s["r"] = (3.0 * normal(M, K)).to(t) if case["residual"] else None
        s["w"] = (1.0 + 0.2 * normal(K)).to(t)
    elif op == "quantize":
        # rows of different size, a few large values in each
        x = normal(case["M"], case["K"]) * torch.exp(normal(case["M"], 1))
        s["x"] = x.to(_TYPES[case["type"]])
    else:
        S, H, A = case["S"], case["H"], case["A"]
        s["x"] = normal(case["M"], S)
        s["layers"] = tuple((*_codes(normal(n, k) / math.sqrt(k)), 0.1 * normal(n)) for n, k in ((H, S), (H, H), (A, H)))
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _plain_act(y, act):
    if act == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if act == "tanh":
        return torch.tanh(y)
    return y


def _plain_linear(q, scale, weight, weight_scale, b, act):
    y = (q.float() @ weight.float().t()) * scale[:, None] * weight_scale
    return _plain_act(y if b is None else y + b, act)


def _plain_quantize(y):
    """Codes (as floating numbers) and scales."""
    top = y.abs().amax(1)
    return torch.round(y * torch.where(top > 0, 127.0 / top, torch.zeros_like(top))[:, None]), top / 127.0


def _plain_norm(x, r, w, eps=1e-6):
    h = x.float() if r is None else x.float() + r.float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + eps) * w.float()
    q, scale = _plain_quantize(y)
    return q, scale, h.to(x.dtype)


def run(s):
    op = s["op"]
    if own:
        from d4pg_pytorch_amd import ops
        if op == "linear":
            return ops.linear_int8(s["q"], s["scale"], s["weight"], s["weight_scale"], s["b"], s["act"], _TYPES[s["type"]])
        if op == "norm":
            q, scale, h = ops.add_rms_norm_int8(s["x"], s["w"], s["r"])
            values = ops.dequantize_rows(q, scale, torch.bfloat16)
            return (values, scale) if s["r"] is None else (values, scale, h)
        if op == "quantize":
            q, scale = ops.quantize_rows(s["x"])
            return ops.dequantize_rows(q, scale, torch.bfloat16), scale
        return ops.mlp3_int8(s["x"], s["layers"], "tanh", torch.bfloat16)
    if op == "linear":
        return _plain_linear(s["q"], s["scale"], s["weight"], s["weight_scale"], s["b"], s["act"]).to(_TYPES[s["type"]])
    if op == "norm":
        q, scale, h = _plain_norm(s["x"], s["r"], s["w"])
        values = (q * scale[:, None]).to(torch.bfloat16)
        return (values, scale) if s["r"] is None else (values, scale, h)
    if op == "quantize":
        q, scale = _plain_quantize(s["x"].float())
        return (q * scale[:, None]).to(torch.bfloat16), scale
    (w1, s1, b1), (w2, s2, b2), (w3, s3, b3) = s["layers"]
    h = _plain_linear(*_plain_quantize(s["x"]), w1, s1, b1, "relu")
    h = _plain_linear(*_plain_quantize(h), w2, s2, b2, "relu")
    return _plain_linear(*_plain_quantize(h), w3, s3, b3, "tanh").to(torch.bfloat16)


# --------------------------------------------------------------------------------------------------- in 64 bits, apart
def _nearest(v):
    """Whole numbers nearest to ``v``, halves to the even one, from floor and comparisons."""
    low = torch.floor(v)
    rest = v - low
    odd = torch.remainder(low, 2.0) == 1.0
    return low + ((rest > 0.5) | ((rest == 0.5) & odd)).to(v.dtype)


def _steps(v):
    """(value each entry of ``v`` [rows, K] stands for after 8 bits, step of each row)."""
    step = torch.maximum(v.max(1, keepdim=True).values, -v.min(1, keepdim=True).values) / 127.0
    safe = torch.where(step == 0.0, torch.ones_like(step), step)
    return _nearest(v / safe) * step, step[:, 0]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = torch.float64

    def layer(values, codes, steps, b):
        y = torch.matmul(values, (codes.to(d) * steps.to(d).unsqueeze(1)).transpose(0, 1))
        return y if b is None else y + b.to(d)

    if op == "linear":
        y = layer(s["q"].to(d) * s["scale"].to(d).unsqueeze(1), s["weight"], s["weight_scale"], s["b"])
        return {"none": lambda v: v, "relu": lambda v: v.clamp_min(0.0), "tanh": torch.tanh}[case["act"]](y)
    if op == "norm":
        h = s["x"].to(d)
        if s["r"] is not None:
            h = h + s["r"].to(d)
        y = h / torch.sqrt(h.square().sum(1, keepdim=True) / case["K"] + 1e-6) * s["w"].to(d)
        values, step = _steps(y)
        return (values, step) if s["r"] is None else (values, step, h)
    if op == "quantize":
        return _steps(s["x"].to(d))
    v = s["x"].to(d)
    for i, (codes, steps, b) in enumerate(s["layers"]):
        v = layer(_steps(v)[0], codes, steps, b)
        v = v.clamp_min(0.0) if i < 2 else torch.tanh(v)
    return v


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    op, M = case["op"], case["M"]
    if op == "policy":
        S, H, A = case["S"], case["H"], case["A"]
        weights = S * H + H * H + H * A
        return {"bytes": 4 * M * S + weights + 8 * (2 * H + A) + 2 * M * A, "flops": 2 * M * weights}
    e = torch.tensor([], dtype=_TYPES[case["type"]]).element_size()
    K = case["K"]
    if op == "linear":
        N = case["N"]
        return {"bytes": M * K + N * K + 4 * (M + N) + (4 * N if case["bias"] else 0) + M * N * e, "flops": 2 * M * N * K}
    if op == "norm":
        # x, the residual and the weight in; codes, scales, what the codes stand for, and the sum out
        return {"bytes": M * K * e * (3 if case["residual"] else 1) + K * e + M * K + 4 * M + 2 * M * K, "flops": 8 * M * K}
    return {"bytes": M * K * e + M * K + 4 * M + 2 * M * K, "flops": 4 * M * K}
