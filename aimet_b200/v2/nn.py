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

Quantized tensors (:mod:`aimet_b200.v2.qtensor`) count as the numbers they hold; results are plain tensors.  There is no
CPU path: CPU tensors raise ``RuntimeError``.  Gradients of gradients and forward-mode derivatives are not provided: both
raise ``RuntimeError``.
"""
from __future__ import annotations

import contextlib
import ctypes
import importlib.util
import os
import threading
from typing import Optional, Sequence, Union

import torch
from torch import nn

from .. import _lib, build

__all__ = ["linear", "layer_norm", "LayerNorm", "ACTIVATIONS", "wait_ran_out"]

#: names the ``activation`` argument takes beside None
ACTIVATIONS = {"relu": _lib.AQ_ACT_RELU, "gelu": _lib.AQ_ACT_GELU, "gelu_tanh": _lib.AQ_ACT_GELU_TANH,
               "silu": _lib.AQ_ACT_SILU}

_ENTRIES = ("aq_status_string", "aq_last_cuda_error", "aq_align_rows", "aq_linear_forward",
            "aq_linear_grad_z_workspace_bytes", "aq_linear_grad_z", "aq_linear_grad_input", "aq_linear_grad_weight",
            "aq_layer_norm_forward", "aq_layer_norm_backward_workspace_bytes", "aq_layer_norm_backward")


def _load():
    """The compiled autograd functions (csrc/torch_layers.cpp), given the entry points of the loaded CUDA library."""
    path = build.TORCH_PATH
    if not os.path.exists(path):
        raise ImportError(f"{path} not found. Build it with `python -m aimet_b200.build`.")
    if build.torch_side_is_foreign(unknown=False):
        raise ImportError(f"{path} was built for another torch or Python. Build it with `python -m aimet_b200.build`.")
    spec = importlib.util.spec_from_file_location("_torch_layers", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.bind({name: ctypes.cast(getattr(_lib.lib, name), ctypes.c_void_p).value for name in _ENTRIES})
    return module


_loading = threading.Lock()


def __getattr__(name):
    # `_layers` is loaded at its first use: a simulated model whose layers are never fused does not need it
    if name != "_layers":
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    with _loading:
        if "_layers" not in globals():
            globals()["_layers"] = _load()
    return globals()["_layers"]


def _native():
    return globals().get("_layers") or __getattr__("_layers")


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    :param x: ``[..., in_features]``, float32, float16 or bfloat16, any strides
    :param weight: ``[out_features, in_features]``, same dtype
    :param bias: ``[out_features]`` or None
    :param activation: None, ``"relu"``, ``"gelu"``, ``"gelu_tanh"`` or ``"silu"``
    :param residual: ``[..., out_features]``, exactly the result's shape (it is not broadcast), or None
    """
    act = _lib.AQ_ACT_NONE
    if activation is not None:
        act = ACTIVATIONS.get(activation)
        if act is None:
            raise ValueError(f"activation must be None or one of {tuple(ACTIVATIONS)}, got {activation!r}")
    return _native().linear(x, weight, bias, act, residual)


def layer_norm(x: torch.Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the trailing dimensions ``normalized_shape``.

    ``x`` is float32, float16 or bfloat16 with any strides; ``weight`` and ``bias``, each optional, have the shape
    ``normalized_shape`` and the dtype of ``x``."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else normalized_shape
    return _native().layer_norm(x, shape, weight, bias, eps)


def wait_ran_out(device: Optional[torch.device] = None) -> bool:
    """Whether a kernel of this module has given up waiting for its own copies or products on ``device`` (default: the
    current one) since the library was loaded.  Every such wait is bounded (4 s); results that a wait was for hold NaN and
    no call fails, so a program that meets NaN asks here.  Waits for the device."""
    out = ctypes.c_int32(0)
    with contextlib.nullcontext() if device is None else torch.cuda.device(device):
        _lib.check(_lib.lib.aq_layers_stuck(ctypes.byref(out)), "aq_layers_stuck")
    return bool(out.value)


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
