"""The layers between the quantizers of a simulated model, as kernels: ``linear`` with bias, activation and residual
fused into the product, ``layer_norm``, both with their backward passes, and the modules that use them.

The reference's quantized layers (aimet_torch/v2/nn/fake_quant.py: ``FakeQuantizedLinear``,
``FakeQuantizedLayerNorm``; parameter handling in v2/nn/base.py:90-196) call torch's own functions between their
quantizers.  :meth:`aimet_b200.v2.quantsim.QuantizationSimModel.fuse_layers` puts the modules below in the place of
the plain ones.

Products and sums are float32 whatever the tensors' dtype; every result is rounded once.  For float16 and bfloat16 the
backward pass works from two rounded intermediates: ``z``, what the activation is applied to, and ``dz``, the gradient
that the two products of the backward pass read -- the tensor cores take operands of the storage type, and a float32
copy would double the traffic.

There is no CPU path: CPU tensors raise ``RuntimeError``.  Gradients of gradients are not provided.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .. import ops
from .._lib import AQ_LINEAR_FEW_ROWS

__all__ = ["linear", "layer_norm", "LayerNorm", "ACTIVATIONS"]

#: names the ``activation`` argument takes beside None
ACTIVATIONS = ("relu", "gelu", "gelu_tanh", "silu")


def _plain(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Quantized tensors count as the numbers they hold."""
    return t if t is None or type(t) is torch.Tensor else t.as_subclass(torch.Tensor)


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` as a matrix of rows of ``width`` elements: a view where rows have unit stride and one pitch."""
    if t.dim() == 2 and t.shape[1] == width:
        m = t
    else:
        try:
            m = t.view(-1, width) if t.numel() else t.reshape(math.prod(t.shape) // max(width, 1), width)
        except RuntimeError:
            m = t.reshape(-1, width)
    if (width > 1 and m.stride(1) != 1) or (m.shape[0] > 1 and m.stride(0) < width):
        m = m.contiguous()
    return m


def _check_operand(t: Optional[torch.Tensor], like: torch.Tensor, shape: tuple, name: str) -> None:
    if t is None:
        return
    if t.shape != shape:
        raise RuntimeError(f"aimet_b200: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    ops._cuda(t, name)   # pylint: disable=protected-access
    if t.dtype is not like.dtype:
        raise RuntimeError(f"aimet_b200: {name} is {t.dtype}, the input is {like.dtype}")
    if t.get_device() != like.get_device():
        ops._same_device(like, t)   # pylint: disable=protected-access


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---------------------------------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------------------------------
def _new_rows(like: torch.Tensor, m: int, n: int) -> torch.Tensor:
    """Uninitialised [m, n] whose rows the tensor cores can read."""
    return like.new_empty((m, n)) if n % 8 == 0 else like.new_empty((m, (n + 7) // 8 * 8))[:, :n]


def _linear_forward(x, weight, bias, residual, activation, keep_z):
    n, k = weight.shape
    xm, wm = _rows(x, k), _rows(weight, k)
    if xm.shape[0] > AQ_LINEAR_FEW_ROWS:
        xm, wm = ops.aligned_rows(xm), ops.aligned_rows(wm)
    rm = None if residual is None else _rows(residual, n)
    bias = None if bias is None else bias.contiguous()
    m = xm.shape[0]
    ym = x.new_empty((m, n))
    z = _new_rows(x, m, n) if keep_z else None
    if m:
        ops.linear_forward(xm, wm, bias, rm, activation, ym, z)
    return ym if x.dim() == 2 else ym.view(x.shape[:-1] + (n,)), z, xm, wm


class _LinearFn(torch.autograd.Function):
    """Keeps x, W (their aligned copies where those were made) and, with an activation, z."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, z, xm, wm = _linear_forward(x, weight, bias, residual, activation, activation is not None)
        ctx.activation = activation
        ctx.x_shape = x.shape
        need_x, need_w = ctx.needs_input_grad[:2]
        ctx.save_for_backward(xm if need_w else None, wm if need_x else None, z)
        ctx.geometry = (xm.shape[0], weight.shape[0], weight.shape[1])
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        xm, wm, z = ctx.saved_tensors
        m, n, k = ctx.geometry
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy = _rows(_plain(grad), n)
        dx = dw = db = None
        if need_b:
            db = dy.new_empty(n)
        dz = dy
        if ctx.activation is not None and (need_x or need_w):
            dz = _new_rows(dy, m, n)
        if need_b or dz is not dy:
            ops.linear_grad_z(dy, z, ctx.activation, None if dz is dy else dz, db)
        if need_x or need_w:
            dz = ops.aligned_rows(dz)
        if need_x:
            dx = dy.new_empty((m, k))
            if m:
                ops.linear_grad_input(dz, ops.aligned_rows(wm), dx)
            if len(ctx.x_shape) != 2:
                dx = dx.view(ctx.x_shape)
        if need_w:
            dw = dy.new_empty((n, k))
            ops.linear_grad_weight(dz, ops.aligned_rows(xm), dw)
        return dx, dw, db, grad if need_r else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    :param x: ``[..., in_features]``, float32, float16 or bfloat16, any strides
    :param weight: ``[out_features, in_features]``, same dtype
    :param bias: ``[out_features]`` or None
    :param activation: None, ``"relu"``, ``"gelu"``, ``"gelu_tanh"`` or ``"silu"``
    :param residual: ``[..., out_features]``, exactly the result's shape (it is not broadcast), or None
    """
    x, weight, bias, residual = _plain(x), _plain(weight), _plain(bias), _plain(residual)
    ops._cuda(x, "input")   # pylint: disable=protected-access
    ops._dt(x)   # pylint: disable=protected-access
    if activation is not None and activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None or one of {ACTIVATIONS}, got {activation!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or not weight.numel():
        raise RuntimeError(f"aimet_b200: cannot apply a weight of shape {tuple(weight.shape)} to an input of shape "
                           f"{tuple(x.shape)}")
    n = weight.shape[0]
    _check_operand(weight, x, weight.shape, "weight")
    _check_operand(bias, x, (n,), "bias")
    _check_operand(residual, x, x.shape[:-1] + (n,), "residual")
    if _wants_grad(x, weight, bias, residual):
        return _LinearFn.apply(x, weight, bias, residual, activation)
    return _linear_forward(x, weight, bias, residual, activation, False)[0]


# ---------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------
def _norm_forward(x, dim, weight, bias, eps, keep_stats):
    xm = _rows(x, dim)
    rows = xm.shape[0]
    y = x.new_empty(x.shape)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    stats, mean, rstd = None, None, None
    if keep_stats:
        stats = x.new_empty((2, rows), dtype=torch.float32)
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    if rows:
        ops.layer_norm_forward(xm, w, b, eps, y, mean, rstd)
    return y, xm, w, stats


class _LayerNormFn(torch.autograd.Function):
    """Keeps x and the mean and reciprocal deviation of every row."""

    @staticmethod
    def forward(ctx, x, weight, bias, shape, eps):
        y, xm, w, stats = _norm_forward(x, math.prod(shape), weight, bias, eps, True)
        ctx.x_shape, ctx.w_shape = x.shape, shape
        ctx.save_for_backward(xm, w, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        xm, w, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = _rows(_plain(grad), xm.shape[1])
        dx = dy.new_empty(ctx.x_shape) if need_x else None
        dw = dy.new_empty(ctx.w_shape) if need_w else None
        db = dy.new_empty(ctx.w_shape) if need_b else None
        mean = stats.data_ptr()
        ops.layer_norm_backward(xm, dy, w, mean, mean + 4 * xm.shape[0], dx, dw, db)
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the trailing dimensions ``normalized_shape``.

    ``x`` is float32, float16 or bfloat16 with any strides; ``weight`` and ``bias``, each optional, have the shape
    ``normalized_shape`` and the dtype of ``x``."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    x, weight, bias = _plain(x), _plain(weight), _plain(bias)
    ops._cuda(x, "input")   # pylint: disable=protected-access
    ops._dt(x)   # pylint: disable=protected-access
    dim = math.prod(shape)
    if not shape or dim < 1 or tuple(x.shape[-len(shape):]) != shape:
        raise RuntimeError(f"aimet_b200: cannot normalise an input of shape {tuple(x.shape)} over {shape}")
    if not 0 <= eps < math.inf:
        raise RuntimeError(f"aimet_b200: eps must be finite and at least 0, got {eps}")
    _check_operand(weight, x, shape, "weight")
    _check_operand(bias, x, shape, "bias")
    if _wants_grad(x, weight, bias):
        return _LayerNormFn.apply(x, weight, bias, shape, eps)
    return _norm_forward(x, dim, weight, bias, eps, False)[0]


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` (parameters, state dict) on :func:`layer_norm`."""

    @classmethod
    def from_module(cls, module: nn.LayerNorm) -> "LayerNorm":
        """Shares the parameters of ``module``."""
        new = cls(module.normalized_shape, module.eps, elementwise_affine=False)
        new.elementwise_affine = module.elementwise_affine
        new.weight, new.bias = module.weight, module.bias
        return new.train(module.training)

    def forward(self, x: torch.Tensor) -> torch.Tensor:   # pylint: disable=arguments-renamed
        return layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps)
