"""Float64 forms of the layer operators and what rounding may add to them.

Bounds, element by element, for operands of type T with half step u (2^-8, 2^-11, 2^-24):

* a float32 sum of n products is off by at most (n + 8) 2^-23 of the sum of their magnitudes: every addition may lose
  one step of 2^-23 (tensor cores cut instead of rounding), the 8 covers bias, residual and the function's own steps;
* a result in T is off by u of its value; its smallest step (subnormals) is added;
* act' is at most 1.13, act'' at most 1.2 for the smooth activations (0.8 for gelu, 0.5 for silu), and gelu, silu, tanh
  and erf come out within 16 steps of 2^-24 of max(1, |z|);
* the backward pass reads z and dz rounded to T.
"""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
F32 = 2.0 ** -23
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def act(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if kind == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, kind):
    if kind is None:
        return torch.ones_like(z)
    zz = z.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(act(zz, kind).sum(), zz)[0]


def linear_ref(x, w, b, r, kind, dy=None):
    """name -> (value, bound) in float64 for matrices x [m, k], w [n, k]."""
    t = x.dtype
    u, tiny = U[t], TINY[t]
    d = lambda v: None if v is None else v.detach().double()   # noqa: E731
    x, w, b, r, dy = d(x), d(w), d(b), d(r), d(dy)
    k, n = x.shape[1], w.shape[0]
    z = x @ w.t()
    ez = (k + 8) * F32 * (x.abs() @ w.abs().t() + (0 if b is None else b.abs()))
    if b is not None:
        z = z + b
    y = act(z, kind)
    ey = 1.13 * ez + (16 * 2.0 ** -24 * z.abs().clamp_min(1) if kind else 0)
    if r is not None:
        y = y + r
        ey = ey + F32 * (y.abs() + r.abs())
    out = {"y": (y, ey * (1 + u) + u * y.abs() + tiny)}
    if dy is None:
        return out
    dz = dy * slope(z, kind)
    if kind is None:
        edz = torch.zeros_like(dz)
    else:
        dev = ez + u * (z.abs() + ez) + tiny             # z as the backward pass reads it
        if kind == "relu":
            eslope = (z.abs() <= dev).double()           # either side of the corner
        else:
            eslope = 1.2 * dev + 32 * 2.0 ** -24
        edz = dy.abs() * eslope + F32 * dz.abs()
    db = dz.sum(0)
    edb = edz.sum(0) + (dz.shape[0] + 8) * F32 * dz.abs().sum(0)
    out["db"] = (db, edb * (1 + u) + u * db.abs() + tiny)
    if kind is not None:
        edz = edz + u * (dz.abs() + edz) + tiny          # dz as the products read it
    adz = dz.abs() + edz
    dx = dz @ w
    edx = edz @ w.abs() + (n + 8) * F32 * (adz @ w.abs())
    out["dx"] = (dx, edx * (1 + u) + u * dx.abs() + tiny)
    dw = dz.t() @ x
    edw = edz.t() @ x.abs() + (x.shape[0] + 8) * F32 * (adz.t() @ x.abs())
    out["dw"] = (dw, edw * (1 + u) + u * dw.abs() + tiny)
    return out


def norm_ref(x, w, b, eps, dy=None):
    """name -> (value, bound) in float64 for x [rows, dim]."""
    t = x.dtype
    u, tiny = U[t], TINY[t]
    x = x.detach().double()
    dim = x.shape[1]
    w = torch.ones(dim, dtype=torch.float64, device=x.device) if w is None else w.detach().double().reshape(-1)
    b = torch.zeros(dim, dtype=torch.float64, device=x.device) if b is None else b.detach().double().reshape(-1)
    g1 = (dim + 8) * 2.0 ** -24
    mu = x.mean(1, keepdim=True)
    c = x - mu
    var = (c * c).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = c * rstd
    emu = g1 * x.abs().mean(1, keepdim=True) + 2.0 ** -24 * mu.abs()
    ec = emu + 2.0 ** -24 * (c.abs() + emu)
    # variance: the sum's own rounding, and every difference off by ec
    evar = 2 * g1 * var + (2 * c.abs() * ec + ec * ec).mean(1, keepdim=True) * (1 + 2 * g1)
    rel = 0.5 * evar / (var + eps) + 4 * 2.0 ** -24
    rel = rel / (1 - 2 * rel).clamp_min(0.25)
    eh = ec * rstd * (1 + rel) + h.abs() * (rel + 2 * 2.0 ** -24)
    y = h * w + b
    ey = eh * w.abs() + 2.0 ** -23 * ((h * w).abs() + b.abs())
    out = {"y": (y, ey * (1 + u) + u * y.abs() + tiny)}
    if dy is None:
        return out
    dy = dy.detach().double()
    g = dy * w
    mg, mgh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    eg = 2.0 ** -24 * g.abs()
    emg = eg.mean(1, keepdim=True) + g1 * g.abs().mean(1, keepdim=True)
    emgh = (g.abs() * eh + eg * h.abs()).mean(1, keepdim=True) + 2 * g1 * (g * h).abs().mean(1, keepdim=True)
    inner = g - mg - h * mgh
    mag = g.abs() + mg.abs() + (h * mgh).abs()
    einner = eg + emg + eh * mgh.abs() + h.abs() * emgh + eh * emgh + 4 * 2.0 ** -24 * mag
    dx = rstd * inner
    edx = rstd * einner * (1 + rel) + dx.abs() * (rel + 2.0 ** -23)
    out["dx"] = (dx, edx * (1 + u) + u * dx.abs() + tiny)
    n = x.shape[0]
    dw, db = (dy * h).sum(0), dy.sum(0)
    edw = (dy.abs() * eh).sum(0) + (n + 8) * 2.0 ** -24 * (dy * h).abs().sum(0)
    edb = (n + 8) * 2.0 ** -24 * dy.abs().sum(0)
    out["dw"] = (dw, edw * (1 + u) + u * dw.abs() + tiny)
    out["db"] = (db, edb * (1 + u) + u * db.abs() + tiny)
    return out


def assert_within(got, ref, what=""):
    want, bound = ref
    got = got.detach().double().reshape(want.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = (got - want).abs() - bound
    if got.numel() and float(over.max()) > 0:
        i = int(over.reshape(-1).argmax())
        raise AssertionError(f"{what}: element {i} is {float(got.reshape(-1)[i])!r}, want {float(want.reshape(-1)[i])!r} "
                             f"within {float(bound.reshape(-1)[i]):.3g}; {int((over > 0).sum())} of {got.numel()} are off")


def norm_error(got, want):
    """||got - want|| / ||want|| in float64."""
    want = want.double()
    return float((got.detach().double().reshape(want.shape) - want).norm() / want.norm())


def float32_norm_bound(depth):
    """What rounding leaves of a float32 sum of ``depth`` products of independent numbers around 0, over its norm.

    After j products the sum is about sqrt(j) products large; rounding it is off by at most 2^-24 of that, with either sign:
    sqrt(sum of j) = depth / sqrt(2) of them against sqrt(depth), so sqrt(depth / 2) 2^-24.  sqrt(depth) leaves room for
    products that share a rounding; 4 more for the last steps.  Operands rounded to 10 bits are off by about 2^-12 each, for
    every depth."""
    return (math.sqrt(depth) + 4) * 2.0 ** -24


FLOAT32_SIZES = [   # m, k, n: one row, few, 32-row tiles, 64 x 64, 128 x 128, with and without a split depth
    (1, 4096, 512), (2, 64, 64), (8, 1000, 333), (31, 2048, 333), (65, 1001, 130), (200, 4000, 96), (128, 2048, 1000),
    (512, 768, 768), (1100, 600, 1544), (1024, 1024, 1024)]
