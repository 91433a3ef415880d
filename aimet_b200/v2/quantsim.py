"""Quantization simulation of a whole model: which tensors get a quantizer, and the calibration driver.

Orchestration only, no arithmetic: every quantizer is a :class:`aimet_b200.v2.quantizer.QuantizeDequantize`.
Mirrors the user-facing surface of ``QuantizationSimModel`` (aimet_torch/v2/quantsim/quantsim.py:71-224: constructor
arguments ``model, dummy_input, quant_scheme, default_output_bw, default_param_bw``; ``sim.model``;
``sim.compute_encodings(forward_pass_callback, forward_pass_callback_args)``) and of the quantized layers
(aimet_torch/v2/nn/base.py:90-196: ``param_quantizers``, ``_compute_param_encodings``).

The reference decides quantizer placement from a JSON configuration and a connected graph of the model; here the
model is traced with ``torch.fx`` and the placement follows the reference's default configuration in its common
form: parameters of convolution / linear layers per output channel, symmetric; the model input, and the output of
every convolution, linear layer, element-wise addition, ReLU and pooling call, asymmetric, per tensor -- except that
a layer or addition whose only consumer is a ReLU is quantized after the ReLU (the "supergroup" rule).  Batch norms
directly after a convolution are folded into it first.
"""
from __future__ import annotations

import contextlib
import copy
import operator
import types
from typing import Callable, Dict, List, Optional

import torch
import torch.nn.functional as F
from torch import fx, nn

from . import nn as qnn
from .encoding_analyzer import MinMaxEncodingAnalyzer, SqnrEncodingAnalyzer, TfEnhancedEncodingAnalyzer
from .quantizer import QuantizeDequantize

__all__ = ["QuantizationSimModel", "QuantizedLayer", "QuantizedLinear", "fold_batch_norms", "fuse_layers"]

_LAYERS = (nn.Conv1d, nn.Conv2d, nn.Conv3d, nn.Linear)
_RELUS = (nn.ReLU, nn.ReLU6)
_POOLS = (nn.MaxPool2d, nn.AvgPool2d, nn.AdaptiveAvgPool2d)
_ADDS = (operator.add, operator.iadd, torch.add)
_RELU_FUNCS = (F.relu, torch.relu, F.relu6)


class QuantizedLayer(nn.Module):
    """A convolution / linear layer whose weight passes through a quantizer on every call
    (the fake-quantized layers of aimet_torch/v2/nn/fake_quant.py; parameter handling of v2/nn/base.py:117-196)."""

    def __init__(self, layer: nn.Module, weight_quantizer: Optional[QuantizeDequantize]):
        super().__init__()
        self.layer = layer
        self.param_quantizers = nn.ModuleDict({"weight": weight_quantizer})

    def forward(self, x):
        wq = self.param_quantizers["weight"]
        if wq is None:
            return self.layer(x)
        return torch.func.functional_call(self.layer, {"weight": wq(self.layer.weight)}, (x,))

    @torch.no_grad()
    def compute_param_encodings(self):
        """Weights are calibrated from the weights themselves, once (base.py:128-150)."""
        wq = self.param_quantizers["weight"]
        if wq is not None:
            with wq.compute_encodings():
                wq(self.layer.weight)


class QuantizedLinear(QuantizedLayer):
    """A linear layer on :func:`aimet_b200.v2.nn.linear`: the activation and the addition that follow it in the traced
    graph arrive as arguments and run in the product's epilogue."""

    def forward(self, x, residual=None, activation=None):   # pylint: disable=arguments-differ
        wq = self.param_quantizers["weight"]
        weight = self.layer.weight if wq is None else wq(self.layer.weight)
        if residual is None:
            return qnn.linear(x, weight, self.layer.bias, activation)
        if isinstance(residual, torch.Tensor) and residual.shape == x.shape[:-1] + weight.shape[:1] and \
                residual.dtype == x.dtype and residual.device == x.device:
            return qnn.linear(x, weight, self.layer.bias, activation, residual)
        return qnn.linear(x, weight, self.layer.bias, activation) + residual   # broadcast or promoted by torch


@torch.no_grad()
def fold_batch_norms(gm: fx.GraphModule) -> int:
    """Folds every BatchNorm that directly follows a convolution (its only consumer) into that convolution:
    W' = W * g / sqrt(var + eps), b' = beta + (b - mean) * g / sqrt(var + eps).  Returns the number folded."""
    mods = dict(gm.named_modules())
    folded = 0
    for node in list(gm.graph.nodes):
        if node.op != "call_module" or not isinstance(mods.get(node.target), (nn.BatchNorm1d, nn.BatchNorm2d)):
            continue
        src = node.args[0]
        if not (isinstance(src, fx.Node) and src.op == "call_module" and isinstance(mods.get(src.target), _LAYERS[:3])
                and len(src.users) == 1):
            continue
        conv, bn = mods[src.target], mods[node.target]
        if bn.training or bn.running_var is None:
            continue
        inv = (bn.weight if bn.weight is not None else torch.ones_like(bn.running_var)) / torch.sqrt(bn.running_var + bn.eps)
        conv.weight.mul_(inv.reshape([-1] + [1] * (conv.weight.dim() - 1)))
        bias = conv.bias if conv.bias is not None else torch.zeros_like(bn.running_mean)
        new_bias = (bias - bn.running_mean) * inv + (bn.bias if bn.bias is not None else 0)
        conv.bias = nn.Parameter(new_bias)
        node.replace_all_uses_with(src)
        gm.graph.erase_node(node)
        folded += 1
    gm.graph.lint()
    gm.recompile()
    gm.delete_all_unused_submodules()
    return folded


def _is_relu(node: fx.Node, mods: Dict[str, nn.Module]) -> bool:
    if node.op == "call_module":
        return isinstance(mods.get(node.target), _RELUS)
    if node.op == "call_function":
        return node.target in _RELU_FUNCS
    return node.op == "call_method" and node.target in ("relu", "relu_")


def _has_hooks(module: nn.Module) -> bool:
    return bool(module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or   # pylint: disable=protected-access
                module._backward_pre_hooks)   # pylint: disable=protected-access


def _activation_name(node: fx.Node, mods: Dict[str, nn.Module]) -> Optional[str]:
    """The epilogue activation that a call node stands for, or None."""
    if node.op == "call_module":
        m = mods.get(node.target)
        if m is None or _has_hooks(m):
            return None
        if type(m) is nn.ReLU:
            return "relu"
        if type(m) is nn.SiLU:
            return "silu"
        if type(m) is nn.GELU:
            return {"none": "gelu", "tanh": "gelu_tanh"}.get(m.approximate)
        return None
    if node.op == "call_method":
        return "relu" if node.target in ("relu", "relu_") else None
    if node.op != "call_function":
        return None
    if node.target in (F.relu, torch.relu, torch.relu_):
        return "relu"
    if node.target is F.silu:
        return "silu"
    if node.target is F.gelu:
        return {"none": "gelu", "tanh": "gelu_tanh"}.get(node.kwargs.get("approximate", "none"))
    return None


_IN_PLACE_FUNCS = (operator.iadd, operator.isub, operator.imul, operator.itruediv, operator.ifloordiv, operator.imod,
                   operator.ipow, operator.iand, operator.ior, operator.ixor, operator.ilshift, operator.irshift,
                   operator.imatmul, operator.setitem)


def _writes_in_place(node: fx.Node, mods: Dict[str, nn.Module]) -> bool:
    if node.op == "call_module":
        m = mods.get(node.target)
        return bool(getattr(m, "inplace", False)) or (m is not None and _has_hooks(m))   # a hook is the user's own code
    if node.op == "call_method":
        return node.target.endswith("_")
    if node.op == "call_function":
        if isinstance(node.target, types.FunctionType) and \
                (node.target.__module__ or "").partition(".")[0] not in ("torch", __name__.partition(".")[0]):
            return True   # the same for torch.fx.wrap
        return (node.target in _IN_PLACE_FUNCS or getattr(node.target, "__name__", "").endswith("_") or
                bool(node.kwargs.get("inplace")) or "out" in node.kwargs or
                any(a is True for a in node.args[1:]))   # F.relu(x, True) and the like
    return False


def _single_user(node: fx.Node) -> Optional[fx.Node]:
    return next(iter(node.users)) if len(node.users) == 1 else None


def fuse_layers(gm: fx.GraphModule) -> int:
    """Puts the linear layers and layer norms of a traced model on the kernels of :mod:`aimet_b200.v2.nn`.

    A quantized ``nn.Linear`` becomes a :class:`QuantizedLinear`; a ReLU, GELU or SiLU that is its only consumer, and
    an addition of another tensor that is the only consumer of the result, move into its epilogue.  Whatever stands
    between them -- an activation quantizer, a second consumer, a module with hooks, a write in place -- keeps them apart,
    so the placement of quantizers and what they see stay as they were.  ``nn.LayerNorm`` modules and ``F.layer_norm`` calls
    are replaced too.  Returns the number of graph nodes that were replaced or taken in."""
    mods = dict(gm.named_modules())
    changed = 0
    for node in list(gm.graph.nodes):
        if node.op == "call_function" and node.target is F.layer_norm and "cudnn_enable" not in node.kwargs and \
                len(node.args) <= 5:
            kw = dict(node.kwargs)
            if "input" in kw:
                kw["x"] = kw.pop("input")
            node.target, node.kwargs = qnn.layer_norm, kw
            changed += 1
        if node.op != "call_module":
            continue
        m = mods.get(node.target)
        if type(m) is nn.LayerNorm and not _has_hooks(m):
            new = qnn.LayerNorm.from_module(m)
        elif type(m) is QuantizedLayer and type(m.layer) is nn.Linear and not _has_hooks(m) and not _has_hooks(m.layer):
            new = QuantizedLinear(m.layer, None)
            new.param_quantizers = m.param_quantizers
            new.train(m.training)
        else:
            continue
        for name, other in list(mods.items()):
            if other is m:
                mods[name] = new
        parent_name, _, leaf = node.target.rpartition(".")
        setattr(gm.get_submodule(parent_name) if parent_name else gm, leaf, new)
        changed += 1
    order = {node: i for i, node in enumerate(gm.graph.nodes)}
    writers = [order[node] for node in gm.graph.nodes if _writes_in_place(node, mods)]
    for node in list(gm.graph.nodes):
        if node.op != "call_module" or type(mods.get(node.target)) is not QuantizedLinear or len(node.args) != 1:
            continue
        last = node
        kwargs = dict(node.kwargs)

        def quiet(user):
            """The fused layer runs, and reads its input, at ``user``: nothing may be written in place on the way there,
            except by the activation that has been taken in."""
            return not any(order[node] < w < order[user] and w != order[last] for w in writers)

        user = _single_user(last)
        if "residual" not in kwargs and "activation" not in kwargs and user is not None and \
                user.args and user.args[0] is last:
            name = _activation_name(user, mods)
            if name is not None and quiet(user):
                kwargs["activation"] = name
                last = user
                user = _single_user(last)
        if "residual" not in kwargs and user is not None and user.op == "call_function" and user.target in _ADDS and \
                len(user.args) == 2 and not user.kwargs:
            left, right = user.args
            other = right if left is last else left
            # x += linear(...) writes to x
            if isinstance(other, fx.Node) and other is not last and quiet(user) and \
                    (user.target is not operator.iadd or left is last):
                kwargs["residual"] = other
                last = user
        if last is node:
            continue
        with gm.graph.inserting_before(last):
            new = gm.graph.call_module(node.target, node.args, kwargs)
        order[new] = order[last]
        last.replace_all_uses_with(new)
        for old in (last, *_between(node, last)):
            gm.graph.erase_node(old)
            changed += 1
    gm.graph.lint()
    gm.recompile()
    gm.delete_all_unused_submodules()
    return changed


def _between(first: fx.Node, last: fx.Node) -> List[fx.Node]:
    """The nodes of a chain from ``last`` (exclusive) back to ``first`` (inclusive)."""
    chain, cur = [], first
    while cur is not last:
        chain.append(cur)
        cur = _single_user(cur)
    return chain[::-1]


class QuantizationSimModel:
    """``sim = QuantizationSimModel(model, dummy_input); sim.compute_encodings(callback, args); sim.model(x)``.

    quant_scheme, mapped to analyzers as the reference does (aimet_torch/quantsim_config/builder.py:294-309):

    * ``"post_training_tf"``: min/max for parameters and activations;
    * ``"post_training_tf_enhanced"``: the v2 ``SqnrEncodingAnalyzer`` (histogram + SQNR search) for parameters (one
      histogram per output channel) and activations;
    * ``"post_training_tf_enhanced_libpymo"``: not a reference scheme name -- activations get the v1 / libpymo
      TF-Enhanced analyzer (512-bucket PDF frozen by the first batch) behind the v2 interface, parameters min/max.
    """

    def __init__(self, model: nn.Module, dummy_input=None, quant_scheme: str = "post_training_tf_enhanced",
                 default_output_bw: int = 8, default_param_bw: int = 8, per_channel_quantization: bool = True,
                 fold_bn: bool = True):
        if quant_scheme not in ("post_training_tf_enhanced", "post_training_tf", "post_training_tf_enhanced_libpymo"):
            raise ValueError(f"unsupported quant_scheme {quant_scheme!r}")
        self._scheme = quant_scheme
        self._act_bw, self._param_bw = int(default_output_bw), int(default_param_bw)
        gm = fx.symbolic_trace(copy.deepcopy(model))
        if fold_bn:
            fold_batch_norms(gm)
        mods = dict(gm.named_modules())
        self.layers: Dict[str, QuantizedLayer] = {}
        self.activation_quantizers: Dict[str, QuantizeDequantize] = {}
        self._activation_keys: Dict[str, tuple] = {}
        # ---- parameters ----
        for node in gm.graph.nodes:
            if node.op == "call_module" and isinstance(mods.get(node.target), _LAYERS):
                layer = mods[node.target]
                shape = (layer.weight.shape[0],) + (1,) * (layer.weight.dim() - 1) if per_channel_quantization else ()
                wq = QuantizeDequantize(shape, self._param_bw, True, self._new_analyzer(shape, for_param=True))
                wq.plain_outputs = True
                wrapped = QuantizedLayer(layer, wq)
                self._set_submodule(gm, node.target, wrapped)
                self.layers[node.target] = wrapped
        mods = dict(gm.named_modules())
        # ---- activations ----
        for node in list(gm.graph.nodes):
            if not self._wants_output_quantizer(node, mods):
                continue
            name = "act_q_" + node.name
            q = QuantizeDequantize((), self._act_bw, False, self._new_analyzer(()))
            q.plain_outputs = True
            # where the exported files list this quantizer: a layer's output, or the model input
            self._activation_keys[name] = ((node.name, "input") if node.op == "placeholder" else
                                           (node.target if node.op == "call_module" else node.name, "output"))
            gm.add_submodule(name, q)
            with gm.graph.inserting_after(node):
                new = gm.graph.call_module(name, (node,))
            node.replace_all_uses_with(new)
            new.args = (node,)
            self.activation_quantizers[name] = q
        gm.graph.lint()
        gm.recompile()
        self.model = gm
        if dummy_input is not None:
            ref = dummy_input[0] if isinstance(dummy_input, (tuple, list)) else dummy_input
            self.model.to(ref.device)

    # ---- construction helpers ----------------------------------------------------------------------------------
    def _new_analyzer(self, shape, for_param: bool = False):
        if self._scheme == "post_training_tf_enhanced":
            return SqnrEncodingAnalyzer(shape)
        if self._scheme == "post_training_tf_enhanced_libpymo" and not for_param:
            return TfEnhancedEncodingAnalyzer(shape)
        return MinMaxEncodingAnalyzer(shape)

    @staticmethod
    def _set_submodule(root: nn.Module, target: str, new: nn.Module):
        parent_name, _, leaf = target.rpartition(".")
        parent = root.get_submodule(parent_name) if parent_name else root
        setattr(parent, leaf, new)

    @staticmethod
    def _wants_output_quantizer(node: fx.Node, mods: Dict[str, nn.Module]) -> bool:
        if node.op == "placeholder":
            return True
        only_user_is_relu = len(node.users) == 1 and _is_relu(next(iter(node.users)), mods)
        if node.op == "call_module":
            m = mods.get(node.target)
            if isinstance(m, QuantizedLayer):
                return not only_user_is_relu
            return isinstance(m, _RELUS + _POOLS)
        if node.op == "call_function":
            if node.target in _ADDS:
                return not only_user_is_relu
            return node.target in _RELU_FUNCS
        return _is_relu(node, mods)

    # ---- calibration -------------------------------------------------------------------------------------------
    def quantizers(self) -> List[QuantizeDequantize]:
        return [l.param_quantizers["weight"] for l in self.layers.values()] + list(self.activation_quantizers.values())

    def compute_encodings(self, forward_pass_callback: Callable, forward_pass_callback_args=None):
        """Calibrates every quantizer: weights from the weights, activations from what flows through the model while
        ``forward_pass_callback(sim.model, forward_pass_callback_args)`` runs (quantsim.py:205-224)."""
        for layer in self.layers.values():
            layer.compute_param_encodings()
        with contextlib.ExitStack() as stack:
            for q in self.activation_quantizers.values():
                stack.enter_context(q.compute_encodings())
            with torch.no_grad():
                forward_pass_callback(self.model, forward_pass_callback_args)

    # ---- kernels for the layers ---------------------------------------------------------------------------------
    def fuse_layers(self) -> int:
        """Runs the linear layers and layer norms of ``sim.model`` on the kernels of :mod:`aimet_b200.v2.nn`
        (:func:`fuse_layers`), with float32 sums in another order than torch's.  Quantizers, encodings and parameters
        stay the same objects.  The default placement has a quantizer behind every linear layer except before a ReLU:
        until ``load_encodings(..., partial=False)`` has removed the quantizers that keep a layer, its activation and its
        residual apart, only ReLUs move into the epilogue; call it again afterwards.  From then on the model needs CUDA
        tensors of one dtype per layer, float32, float16 or bfloat16 (no autocast).  Meant for models in 16 bits: float32
        products are slower than torch's."""
        changed = fuse_layers(self.model)
        self.layers = {name: self.model.get_submodule(name) for name in self.layers}
        return changed

    # ---- encodings on disk -------------------------------------------------------------------------------------
    def get_encodings_dict(self) -> dict:
        """The calibrated encodings in the layout of the reference's ``<prefix>_torch.encodings`` file
        (aimet_torch/v1/quantsim.py:884-938, 1028-1040): ``param_encodings`` maps ``<layer>.weight`` to one dict per
        output channel, ``activation_encodings`` maps a layer name to ``{"input" | "output": {"0": dict}}``; every
        dict is what ``get_legacy_encodings`` returns.  Quantizers that were never calibrated are left out."""
        params, acts = {}, {}
        for name, layer in self.layers.items():
            wq = layer.param_quantizers["weight"]
            enc = wq.get_legacy_encodings() if wq is not None else None
            if enc is not None:
                params[name + ".weight"] = enc
        for name, q in self.activation_quantizers.items():
            enc = q.get_legacy_encodings()
            if enc is not None:
                key, kind = self._activation_keys[name]
                acts.setdefault(key, {}).setdefault(kind, {})["0"] = enc[0]
        return {"version": "0.6.1", "activation_encodings": acts, "param_encodings": params, "excluded_layers": []}

    def export_encodings(self, path: str, filename_prefix: str) -> str:
        """Writes ``<path>/<filename_prefix>_torch.encodings`` (JSON) and returns its name."""
        import json
        import os
        os.makedirs(path, exist_ok=True)
        target = os.path.join(path, filename_prefix + "_torch.encodings")
        with open(target, "w") as f:
            json.dump(self.get_encodings_dict(), f, sort_keys=True, indent=4)
        return target

    def load_encodings(self, encodings, strict: bool = True, partial: bool = True,
                       requires_grad: Optional[bool] = None, allow_overwrite: bool = True):
        """Sets quantizers from an encodings dictionary or file (aimet_torch/v1/quantsim.py:1695-1756 with the
        per-layer rules of aimet_torch/v2/nn/base.py:282-420).  ``strict``: unknown names raise; ``partial`` = False:
        quantizers the dictionary does not mention are removed; ``requires_grad``: trainability of the loaded
        ranges (None = unchanged); ``allow_overwrite`` = False freezes them against later calibration.  Quantizers
        that were frozen by an earlier load are skipped."""
        import json
        import os
        if isinstance(encodings, (str, os.PathLike)):
            with open(encodings) as f:
                encodings = json.load(f)
        if "param_encodings" not in encodings:
            params, acts = encodings, {}
        else:
            params, acts = encodings.get("param_encodings", {}), encodings.get("activation_encodings", {})
        if not params and not acts:
            raise RuntimeError("the encodings dictionary is empty")
        by_key = {self._activation_keys[name]: name for name in self.activation_quantizers}
        if strict:
            known = {n + ".weight" for n in self.layers} | {key for key, _ in by_key}
            missing = sorted((set(params) | set(acts)) - known)
            if missing:
                raise RuntimeError("Encoding dictionary contains modules/parameters that doesn't exist in the model: "
                                   + ", ".join(missing))

        def apply(q, enc):
            q.set_legacy_encodings([enc] if isinstance(enc, dict) else list(enc))
            if requires_grad is not None:
                q.requires_grad_(requires_grad)
            q.allow_overwrite(allow_overwrite)

        for name, layer in self.layers.items():
            wq = layer.param_quantizers["weight"]
            if wq is not None and not wq._allow_overwrite:   # pylint: disable=protected-access
                continue
            enc = params.get(name + ".weight")
            if not enc:
                if not partial:
                    layer.param_quantizers["weight"] = None
                continue
            if wq is None:
                if strict:
                    raise RuntimeError(f"Failed to import encoding of {name}.weight: no quantizer present.")
                continue
            apply(wq, enc)
        for (key, kind), name in by_key.items():
            q = self.activation_quantizers[name]
            if not q._allow_overwrite:   # pylint: disable=protected-access
                continue
            enc = acts.get(key, {}).get(kind, {})
            enc = enc.get("0", enc.get(0)) if isinstance(enc, dict) else None
            if not enc:
                if not partial:
                    self._remove_activation_quantizer(name)
                continue
            apply(q, enc)

    def _remove_activation_quantizer(self, name: str):
        """Takes a quantizer out of the traced graph: its consumers read the tensor it used to wrap."""
        for node in list(self.model.graph.nodes):
            if node.op == "call_module" and node.target == name:
                node.replace_all_uses_with(node.args[0])
                self.model.graph.erase_node(node)
        self.model.graph.lint()
        self.model.recompile()
        self.model.delete_submodule(name)
        del self.activation_quantizers[name]
        del self._activation_keys[name]

