"""The layer operators of a quantization simulation's transformer blocks, as cases to be measured.

* ``linear``: ``act(x W^T + b) + r`` and its gradients, the product behind every quantized linear layer;
* ``layer_norm``: the normalisation in front of it and its gradients, the sums over the rows for weight and bias
  among them.

``run`` computes a case in plain torch operations (float32 inside, one rounding at the end) or, with ``own``,
through ``aimet_b200.v2.nn``.  ``exact`` is the definition in float64.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _linear(name, rows, k, n, dtype, activation="none", bias=True, residual=False, train=False, pitched=False):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "activation": activation,
            "bias": bias, "residual": residual, "train": train, "pitched": pitched}


def _norm(name, rows, dim, dtype, train=False, pitched=False):
    return {"name": name, "op": "layer_norm", "rows": rows, "dim": dim, "dtype": dtype, "train": train,
            "pitched": pitched}


def listed():
    return [
        # one new token through the up projection of a decoder layer (hidden 4096, MLP 11008)
        _linear("linear_one_token_bf16", 1, 4096, 11008, "bfloat16", "silu", bias=False),
        # a small batch of tokens through the down projection, added to the residual stream
        _linear("linear_few_tokens_fp16", 24, 11008, 4096, "float16", residual=True),
        # a prompt of 2048 tokens through the up projection
        _linear("linear_prompt_bf16", 2048, 4096, 11008, "bfloat16", "gelu_tanh"),
        # a training step of the down projection; its input is one half of a packed pair of projections
        _linear("linear_train_pitched_bf16", 2048, 11008, 4096, "bfloat16", residual=True, train=True, pitched=True),
        # a training step of the up projection on 8 sequences of 2048 tokens
        _linear("linear_train_bf16", 16384, 4096, 11008, "bfloat16", "gelu", train=True),
        # odd sizes throughout: no row starts on a 16-byte boundary
        _linear("linear_train_ragged_fp16", 777, 1001, 1537, "float16", "relu", residual=True, train=True),
        # the classifier of an image model in single precision, batch of 128
        _linear("linear_train_classifier_fp32", 128, 2048, 1000, "float32", train=True),
        # the normalisation in front of the projections: one token, a prompt, 8 sequences of a training batch
        _norm("norm_one_token_bf16", 1, 4096, "bfloat16"),
        _norm("norm_prompt_bf16", 2048, 4096, "bfloat16"),
        _norm("norm_train_bf16", 16384, 4096, "bfloat16", train=True),
        # odd rows and an odd width in single precision
        _norm("norm_train_ragged_fp32", 5003, 1537, "float32", train=True),
        # wide rows that are a part of wider ones
        _norm("norm_train_wide_fp16", 1024, 11008, "float16", train=True, pitched=True),
    ]


def _spread(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = max(lo, min(hi, v))
    kind = rng.random()
    if kind < 0.5 and v >= 64:
        v -= v % 64          # the multiples that models use
    elif kind < 0.75:
        v |= 1               # odd sizes
    return v


def draw(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    train = rng.random() < 0.5
    pitched = rng.random() < 0.25
    if rng.random() < 0.6:
        cap = 16384 * 4096 * 11008 // (8 if dtype == "float32" else 1)
        while True:
            rows, k, n = _spread(rng, 1, 16384), _spread(rng, 32, 11008), _spread(rng, 32, 11008)
            if rows * k * n <= cap:
                break
        case = _linear("", rows, k, n, dtype, rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                       rng.random() < 0.6, rng.random() < 0.4, train, pitched)
    else:
        while True:
            rows, dim = _spread(rng, 1, 65536), _spread(rng, 8, 16384)
            if rows * dim <= 16384 * 4096:
                break
        case = _norm("", rows, dim, dtype, train, pitched)
    del case["name"]
    return case


def _rows_of(case, width, gen, dtype, scale=1.0, shift=0.0):
    """[rows, width] of normal values; a pitched one is the left part of rows that are 64 elements longer."""
    rows = case["rows"]
    full = width + 64 if case["pitched"] else width
    x = torch.randn(rows, full, device="cuda", generator=gen) * scale + shift
    return x.to(dtype)[:, :width]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    train = case["train"]
    s = {"case": case, "dtype": dtype}
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        s["x"] = _rows_of(case, k, gen, dtype)
        # weights as a fake-quantizer leaves them: 8 bits, symmetric, one scale per output channel
        w = torch.randn(n, k, device="cuda", generator=gen) * (1.0 / math.sqrt(k))
        step = w.abs().amax(dim=1, keepdim=True) / 127
        s["w"] = (torch.round(w / step) * step).to(dtype)
        s["b"] = (torch.randn(n, device="cuda", generator=gen) * 0.1).to(dtype) if case["bias"] else None
        s["r"] = torch.randn(case["rows"], n, device="cuda", generator=gen).to(dtype) if case["residual"] else None
        s["dy"] = torch.randn(case["rows"], n, device="cuda", generator=gen).to(dtype) if train else None
    else:
        dim = case["dim"]
        # a residual stream: a mean of its own and a few channels far larger than the rest
        channel = torch.where(torch.rand(dim, device="cuda", generator=gen) < 0.01, 20.0, 1.0)
        s["x"] = (_rows_of(case, dim, gen, torch.float32, 1.0, 0.25) * channel).to(dtype)
        if case["pitched"]:
            wide = torch.empty(case["rows"], dim + 64, device="cuda", dtype=dtype)
            wide[:, :dim].copy_(s["x"])
            s["x"] = wide[:, :dim]
        s["w"] = (1 + 0.1 * torch.randn(dim, device="cuda", generator=gen)).to(dtype)
        s["b"] = (0.1 * torch.randn(dim, device="cuda", generator=gen)).to(dtype)
        s["dy"] = torch.randn(case["rows"], dim, device="cuda", generator=gen).to(dtype) if train else None
        s["eps"] = 1e-5
    if train:
        for name in ("x", "w", "b", "r"):
            if s.get(name) is not None:
                s[name] = s[name].detach().requires_grad_(True)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _act(z, kind):
    if kind == "relu":
        return torch.clamp_min(z, 0)
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if kind == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_linear(s):
    case, dtype = s["case"], s["dtype"]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    y = _act(z, case["activation"])
    if s["r"] is not None:
        y = y + s["r"].detach().float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        dz = s["dy"].float() * _act_slope(z, case["activation"])
        out["dx"] = (dz @ w).to(dtype)
        out["dw"] = (dz.t() @ x).to(dtype)
        if s["b"] is not None:
            out["db"] = dz.sum(dim=0).to(dtype)
        if s["r"] is not None:
            out["dr"] = s["dy"]
    return out


def _plain_norm(s):
    case, dtype = s["case"], s["dtype"]
    x, w, b = s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    c = x - x.mean(dim=1, keepdim=True)
    r = torch.rsqrt((c * c).mean(dim=1, keepdim=True) + s["eps"])
    h = c * r
    out = {"y": (h * w + b).to(dtype)}
    if case["train"]:
        dy = s["dy"].float()
        g = dy * w
        out["dx"] = (r * (g - g.mean(dim=1, keepdim=True) - h * (g * h).mean(dim=1, keepdim=True))).to(dtype)
        out["dw"] = (dy * h).sum(dim=0).to(dtype)
        out["db"] = dy.sum(dim=0).to(dtype)
    return out


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _own_linear(s):
    from aimet_b200.v2 import nn as qnn
    case = s["case"]
    act = None if case["activation"] == "none" else case["activation"]
    y = qnn.linear(s["x"], s["w"], s["b"], activation=act, residual=s["r"])
    if not case["train"]:
        return {"y": y}
    names = [name for name in ("x", "w", "b", "r") if s[name] is not None]
    grads = torch.autograd.grad(y, [s[name] for name in names], s["dy"])
    return {"y": y.detach(), **{"d" + name: g for name, g in zip(names, grads)}}


def _own_norm(s):
    from aimet_b200.v2 import nn as qnn
    case = s["case"]
    y = qnn.layer_norm(s["x"], (case["dim"],), s["w"], s["b"], eps=s["eps"])
    if not case["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def run(state):
    linear = state["case"]["op"] == "linear"
    if own:
        return _own_linear(state) if linear else _own_norm(state)
    return _plain_linear(state) if linear else _plain_norm(state)


def work(case):
    e = _DTYPES[case["dtype"]].itemsize
    rows, train = case["rows"], case["train"]
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        elements = rows * k + n * k + rows * n          # x, W, y
        elements += n if case["bias"] else 0
        elements += rows * n if case["residual"] else 0
        flops = 2 * rows * k * n
        if train:
            elements += rows * n + rows * k + n * k     # dy, dx, dW (the residual's gradient is dy itself)
            elements += n if case["bias"] else 0
            flops *= 3
        return {"bytes": elements * e, "flops": flops}
    dim = case["dim"]
    elements = 2 * rows * dim + 2 * dim                 # x, y; weight and bias
    flops = 8 * rows * dim
    if train:
        elements += 2 * rows * dim + 2 * dim            # dy, dx; their gradients
        flops += 16 * rows * dim
    return {"bytes": elements * e, "flops": flops}


# ---- the definition in float64, differentiated by autograd -----------------------------------------------------------
def _phi(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def exact(case, seed):
    s = prepare(case, seed)
    leaf = {}
    for name in ("x", "w", "b", "r"):
        if s.get(name) is not None:
            leaf[name] = s[name].detach().double().requires_grad_(case["train"])
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "linear":
            z = torch.matmul(leaf["x"], leaf["w"].transpose(0, 1))
            if "b" in leaf:
                z = z + leaf["b"][None, :]
            kind = case["activation"]
            if kind == "relu":
                y = torch.where(z > 0, z, torch.zeros_like(z))
            elif kind == "gelu":
                y = z * _phi(z)
            elif kind == "gelu_tanh":
                # (1 + tanh u) / 2 is the logistic function of 2u
                y = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
            elif kind == "silu":
                y = z * torch.sigmoid(z)
            else:
                y = z
            if "r" in leaf:
                y = y + leaf["r"]
        else:
            x = leaf["x"]
            mean = x.sum(dim=-1, keepdim=True) / case["dim"]
            var = ((x - mean) ** 2).sum(dim=-1, keepdim=True) / case["dim"]
            y = (x - mean) / torch.sqrt(var + s["eps"]) * leaf["w"] + leaf["b"]
    out = {"y": y.detach()}
    if case["train"]:
        names = list(leaf)
        for name, g in zip(names, torch.autograd.grad(y, [leaf[n] for n in names], s["dy"].double())):
            out["d" + name] = g
    return out
