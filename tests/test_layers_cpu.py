"""Layer operators without a GPU: argument checks of the C entries and of the Python layer, and the graph rewriting."""
import pytest
import torch
from torch import nn
import torch.nn.functional as F


def test_c_entries_reject_bad_arguments():
    from aimet_b200._lib import lib
    p = 1 << 20   # never read: every call below is refused before a launch
    fwd = lambda x=p, ldx=64, w=p, ldw=64, b=None, r=None, ldr=0, y=p, ldy=32, z=None, ldz=0, dt=2, m=9, n=32, k=64, act=0: \
        lib.aq_linear_forward(x, ldx, w, ldw, b, r, ldr, y, ldy, z, ldz, dt, m, n, k, act, None)   # noqa: E731
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(ldx=63), dict(ldw=60), dict(ldy=31), dict(dt=3), dict(dt=-1),
                dict(m=-1), dict(n=0), dict(k=0), dict(act=5), dict(act=-1), dict(x=p + 2), dict(w=p + 8), dict(ldx=68),
                dict(ldw=66), dict(r=p, ldr=31), dict(z=p, ldz=16), dict(b=p + 1), dict(y=p + 1),
                dict(dt=0, x=p + 2), dict(dt=0, r=p + 2, ldr=32)):
        assert fwd(**bad) == -1, bad
    assert fwd(m=1 << 32) == -5 and fwd(n=1 << 32, ldy=1 << 32) == -5
    assert fwd(m=0, x=None, y=None) == 0
    gz = lambda dy=p, z=p, dz=p, db=p, dt=2, m=4, n=32, act=2, ws=p, need=1 << 30: \
        lib.aq_linear_grad_z(dy, 32, z, 32, dz, 32, db, dt, m, n, act, ws, need, None)   # noqa: E731
    for bad in (dict(dy=None), dict(z=None), dict(dt=7), dict(m=-1), dict(n=0), dict(act=9), dict(n=33), dict(db=p + 1)):
        assert gz(**bad) == -1, bad
    assert gz(ws=None) == -4 and gz(ws=p + 128) == -4 and gz(need=16) == -4
    assert gz(m=0, dy=None, z=None, dz=None, db=None) == 0
    for fn, rows in ((lib.aq_linear_grad_input, 0), (lib.aq_linear_grad_weight, 1)):
        call = lambda a=p, lda=32, b=p, ldb=64, o=p, ldo=64, dt=2, m=4, n=32, k=64, fn=fn: \
            fn(a, lda, b, ldb, o, ldo, dt, m, n, k, None)   # noqa: E731
        for bad in (dict(a=None), dict(b=None), dict(o=None), dict(lda=31), dict(ldb=63), dict(ldo=63), dict(dt=4),
                    dict(m=-1), dict(n=0), dict(k=0), dict(a=p + 2), dict(b=p + 4), dict(lda=36), dict(ldb=65)):
            assert call(**bad) == -1, (fn, bad)
        assert call(m=1 << 32) == -5
    assert lib.aq_linear_grad_input(None, 32, p, 64, None, 64, 2, 0, 32, 64, None) == 0
    assert lib.aq_align_rows(p, 7, p, 8, 2, 4, 8, None) == -1 and lib.aq_align_rows(p, 8, p + 2, 8, 2, 4, 8, None) == -1
    assert lib.aq_align_rows(p, 9, p, 9, 1, 4, 9, None) == -1 and lib.aq_align_rows(p, 9, p, 16, 1, -1, 9, None) == -1


def test_c_layer_norm_rejects_bad_arguments():
    from aimet_b200._lib import lib
    p = 1 << 20
    fwd = lambda x=p, ldx=32, w=None, b=None, y=p, mean=None, rstd=None, dt=2, rows=4, dim=32, eps=1e-5: \
        lib.aq_layer_norm_forward(x, ldx, w, b, y, mean, rstd, dt, rows, dim, eps, None)   # noqa: E731
    for bad in (dict(x=None), dict(y=None), dict(ldx=31), dict(mean=p), dict(rstd=p), dict(dt=3), dict(rows=-1), dict(dim=0),
                dict(eps=-1.0), dict(eps=float("nan")), dict(x=p + 1), dict(w=p + 1), dict(dt=0, b=p + 2)):
        assert fwd(**bad) == -1, bad
    assert fwd(rows=1 << 32) == -5 and fwd(rows=0, x=None, y=None) == 0
    bwd = lambda x=p, dy=p, lddy=32, mean=p, rstd=p, dx=p, dw=p, db=p, dt=2, rows=4, dim=32, ws=p, need=1 << 30: \
        lib.aq_layer_norm_backward(x, 32, dy, lddy, None, mean, rstd, dx, dw, db, dt, rows, dim, ws, need, None)   # noqa: E731
    for bad in (dict(x=None), dict(dy=None), dict(mean=None), dict(rstd=None), dict(lddy=31), dict(dt=3), dict(rows=-1),
                dict(dim=0), dict(dim=33), dict(dx=p + 1), dict(dw=p + 1)):
        assert bwd(**bad) == -1, bad
    assert bwd(ws=None) == -4 and bwd(need=8) == -4 and bwd(ws=p + 16) == -4
    assert bwd(rows=0, x=None, dy=None, mean=None, rstd=None, dw=None, db=None) == 0
    assert lib.aq_layer_norm_backward_workspace_bytes(2, 100, 64) > 0
    assert lib.aq_layer_norm_backward_workspace_bytes(2, -1, 64) == -1
    assert lib.aq_linear_grad_z_workspace_bytes(2, 0, 64) > 0 and lib.aq_linear_grad_z_workspace_bytes(9, 4, 64) == -1


def test_python_refuses_cpu_tensors_and_bad_names():
    from aimet_b200.v2.nn import layer_norm, linear
    x, w = torch.randn(2, 8), torch.randn(4, 8)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        linear(x, w)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        layer_norm(x, 8)


def test_rows_views():
    from aimet_b200.v2.nn import _layers
    _rows = _layers.rows_of
    t = torch.randn(4, 6, 8)
    assert _rows(t, 8).data_ptr() == t.data_ptr() and _rows(t, 8).shape == (24, 8)
    s = torch.randn(4, 6, 16)[..., 4:12]
    assert _rows(s, 8).data_ptr() == s.data_ptr() and _rows(s, 8).stride() == (16, 1)
    for odd in (torch.randn(8, 24).t(), torch.randn(1, 8).expand(5, 8), torch.randn(5, 16)[:, ::2],
                torch.randn(40).as_strided((5, 8), (4, 1)), torch.randn(6, 4, 8).transpose(0, 1)):
        m = _rows(odd, 8)
        assert m.stride(1) == 1 and (m.shape[0] == 1 or m.stride(0) >= 8) and torch.equal(m, odd.reshape(-1, 8))
    assert _rows(torch.randn(8), 8).shape == (1, 8)
    assert _rows(torch.empty(3, 0, 8), 8).shape == (0, 8)


@pytest.fixture
def on_torch(monkeypatch):
    """The kernels replaced by torch's own functions, so that rewritten graphs run here; calls are recorded."""
    from aimet_b200.v2 import nn as qnn
    calls = []

    def linear(x, weight, bias=None, activation=None, residual=None):
        calls.append(("linear", activation, residual is not None))
        y = F.linear(x, weight, bias)
        y = {None: lambda v: v, "relu": F.relu, "gelu": F.gelu, "silu": F.silu,
             "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[activation](y)
        return y if residual is None else y + residual

    def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5):
        calls.append(("layer_norm",))
        return F.layer_norm(x, normalized_shape if not isinstance(normalized_shape, int) else (normalized_shape,), weight,
                            bias, eps)

    monkeypatch.setattr(qnn, "linear", linear)
    monkeypatch.setattr(qnn, "layer_norm", layer_norm)
    return calls


def _fused(model):
    """A traced model with bare (unquantized) layers and no activation quantizers, rewritten."""
    from aimet_b200.v2.quantsim import QuantizationSimModel
    sim = QuantizationSimModel(model)
    for layer in sim.layers.values():
        layer.param_quantizers["weight"] = None
    for name in list(sim.activation_quantizers):
        sim._remove_activation_quantizer(name)
    return sim, sim.fuse_layers()


class _Net(nn.Module):
    def __init__(self, fn, **mods):
        super().__init__()
        self.a, self.b, self.n = nn.Linear(8, 8), nn.Linear(8, 8), nn.LayerNorm(8)
        for k, v in mods.items():
            setattr(self, k, v)
        self.fn = fn

    def forward(self, x):
        return self.fn(self, x)


@pytest.mark.parametrize("fn,mods,want", [
    (lambda s, x: s.r(s.a(x)), {"r": nn.ReLU()}, [("linear", "relu", False)]),
    (lambda s, x: s.r(s.a(x)), {"r": nn.ReLU(inplace=True)}, [("linear", "relu", False)]),
    (lambda s, x: s.r(s.a(x)), {"r": nn.ReLU6()}, [("linear", None, False)]),
    (lambda s, x: s.r(s.a(x)), {"r": nn.GELU("tanh")}, [("linear", "gelu_tanh", False)]),
    (lambda s, x: F.gelu(s.a(x)), {}, [("linear", "gelu", False)]),
    (lambda s, x: F.silu(s.a(x)) + x, {}, [("linear", "silu", True)]),
    (lambda s, x: x + s.a(x), {}, [("linear", None, True)]),
    (lambda s, x: torch.add(s.a(x), x), {}, [("linear", None, True)]),
    (lambda s, x: torch.add(s.a(x), x, alpha=2), {}, [("linear", None, False)]),
    (lambda s, x: s.a(x) + 1.5, {}, [("linear", None, False)]),
    (lambda s, x: (lambda y: y + y)(s.a(x)), {}, [("linear", None, False)]),
    (lambda s, x: (lambda y: F.relu(y) + y)(s.a(x)), {}, [("linear", None, False)]),
    (lambda s, x: s.b(F.relu(s.a(s.n(x)))) + x, {}, [("layer_norm",), ("linear", "relu", False), ("linear", None, True)]),
    (lambda s, x: F.layer_norm(s.a(x), (8,), s.n.weight, eps=0.1), {}, [("linear", None, False), ("layer_norm",)]),
    (lambda s, x: s.a(x) + s.b(x), {}, None),
    (lambda s, x: s.a(x) + x[:1], {}, [("linear", None, False)]),
    (lambda s, x: s.a(F.relu(s.a(x))), {}, [("linear", "relu", False), ("linear", None, False)]),
])
def test_fuse_layers_keeps_the_function(on_torch, fn, mods, want):
    torch.manual_seed(0)
    net = _Net(fn, **mods).eval()
    x = torch.randn(5, 8)
    expect = net(x.clone())
    sim, changed = _fused(net)
    assert changed > 0
    assert torch.allclose(sim.model(x.clone()), expect, atol=1e-6)
    if want is not None:
        assert on_torch == want


def test_fuse_layers_leaves_in_place_writes_alone(on_torch):
    """A tensor that is written between the layer that reads it and the addition."""
    def written_between(s, x):
        h = x * 1.0
        y = s.a(h)
        h.mul_(2.0)
        return y + h

    torch.manual_seed(0)
    net = _Net(written_between).eval()
    x = torch.randn(5, 8)
    expect = net(x.clone())
    sim, _ = _fused(net)
    assert torch.allclose(sim.model(x.clone()), expect, atol=1e-6)
    assert on_torch == [("linear", None, False)]


def test_fuse_layers_stops_at_quantizers_and_hooks():
    from aimet_b200.v2.quantsim import QuantizationSimModel, QuantizedLinear
    sim = QuantizationSimModel(_Net(lambda s, x: s.b(F.gelu(s.a(x))) + x))
    names = dict(sim.activation_quantizers)
    wq = {n: l.param_quantizers["weight"] for n, l in sim.layers.items()}
    sim.fuse_layers()
    # quantizers stand between layer, activation and addition: only the layers themselves change
    assert sim.activation_quantizers == names and all(type(l) is QuantizedLinear for l in sim.layers.values())
    assert all(l.param_quantizers["weight"] is wq[n] for n, l in sim.layers.items())
    calls = [n for n in sim.model.graph.nodes if n.op == "call_module" and n.target in ("a", "b")]
    assert all(not n.kwargs and len(n.args) == 1 for n in calls)
    assert "act_q_a" in names and "act_q_b" in names
    hooked = _Net(lambda s, x: s.r(s.a(x)), r=nn.ReLU())
    sim = QuantizationSimModel(hooked)
    for name in list(sim.activation_quantizers):
        sim._remove_activation_quantizer(name)
    sim.model.get_submodule("r").register_forward_hook(lambda *a: None)
    sim.fuse_layers()
    assert any(n.op == "call_module" and n.target == "r" for n in sim.model.graph.nodes)


def test_layer_norm_module_shares_parameters():
    from aimet_b200.v2.nn import LayerNorm
    old = nn.LayerNorm((3, 4), eps=0.1)
    new = LayerNorm.from_module(old.eval())
    assert new.weight is old.weight and new.bias is old.bias and new.eps == 0.1 and not new.training
    assert new.state_dict().keys() == old.state_dict().keys()
    bare = LayerNorm.from_module(nn.LayerNorm(5, elementwise_affine=False))
    assert bare.weight is None and bare.bias is None


def _mul_between(s, x):
    h = x * 1.0
    y = s.a(h)
    h.mul_(2.0)
    return F.relu(y)


def _relu_between(s, x):
    h = x * 1.0
    y = s.a(h)
    h.relu_()
    return F.gelu(y) + s.b(h)


def _module_between(s, x):
    h = s.n(x)
    y = s.a(h)
    g = s.r(h)
    return F.silu(y) * g


def _function_between(s, x):
    h = x * 1.0
    y = s.a(h)
    F.relu(h, inplace=True)
    return torch.relu(y)


def _dropout_between(s, x):
    h = x * 1.0
    y = s.a(h)
    F.dropout(h, 1.0, True, inplace=True)
    return s.g(y)


def _between_activation_and_addition(s, x):
    h = x * 1.0
    y = F.relu(s.a(h))
    h.mul_(2.0)
    return y + x


@torch.fx.wrap
def _doubled(h):
    return h.mul_(2.0)


def _wrapped_function_between(s, x):
    h = x * 1.0
    y = s.a(h)
    g = _doubled(h)
    return F.relu(y) * g


@pytest.mark.parametrize("fn,mods,want", [
    (_mul_between, {}, [("linear", None, False)]),
    (_relu_between, {}, None),
    (_module_between, {"r": nn.ReLU(inplace=True)}, [("layer_norm",), ("linear", None, False)]),
    (_function_between, {}, [("linear", None, False)]),
    (_dropout_between, {"g": nn.GELU()}, [("linear", None, False)]),
    (_between_activation_and_addition, {}, [("linear", "relu", False)]),
    (_wrapped_function_between, {}, [("linear", None, False)]),
])
def test_fuse_layers_reads_the_input_before_it_is_written(on_torch, fn, mods, want):
    """The layer's input is written in place before the activation (or the addition) is reached."""
    torch.manual_seed(0)
    net = _Net(fn, **mods).eval()
    x = torch.randn(5, 8)
    expect = net(x.clone())
    sim, _ = _fused(net)
    assert torch.allclose(sim.model(x.clone()), expect, atol=1e-6)
    if want is not None:
        assert on_torch == want


def test_forward_mode_tensors_are_refused():
    """A result without a tangent would be taken for a constant."""
    import torch.autograd.forward_ad as fwad
    from aimet_b200.v2.nn import layer_norm, linear
    x, w, b = torch.randn(2, 8), torch.randn(4, 8), torch.randn(4)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))   # noqa: E731
        for call in (lambda: linear(dual(x), w), lambda: linear(x, dual(w)), lambda: linear(x, w, dual(b)),
                     lambda: linear(x, w, residual=dual(torch.zeros(2, 4))), lambda: layer_norm(dual(x), 8),
                     lambda: layer_norm(x, 8, dual(torch.ones(8))), lambda: layer_norm(x, 8, None, dual(torch.ones(8)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with torch.inference_mode(), pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            linear(dual(x), w)   # no tangents are carried here, by torch's functions neither


def test_rows_of_lazily_negated_tensors():
    from aimet_b200.v2.nn import _layers
    for t in (torch.randn(4, 8), torch.randn(2, 3, 8), torch.randn(8)):
        n = torch._neg_view(t)
        rows = _layers.rows_of(n, 8)
        assert n.is_neg() and not rows.is_neg() and torch.equal(rows, -t.reshape(-1, 8))


def test_wait_ran_out_asks_the_library(monkeypatch):
    """A library that answers as one whose wait has run out, as a sound one, and as one that cannot be asked."""
    from aimet_b200.v2 import nn as qnn
    real = qnn._lib.lib
    answers = iter([(0, 1), (0, 0), (-3, 0)])

    class Fake:
        def aq_layers_stuck(self, out):
            rc, out._obj.value = next(answers)
            return rc

        def __getattr__(self, name):
            return getattr(real, name)

    monkeypatch.setattr(qnn._lib, "lib", Fake())
    assert qnn.wait_ran_out() is True
    assert qnn.wait_ran_out() is False
    with pytest.raises(RuntimeError, match="aq_layers_stuck"):
        qnn.wait_ran_out()


def test_simulated_models_do_not_need_the_torch_side():
    """Without _torch_layers.so everything but the two layers works; these say what is missing."""
    import os
    import subprocess
    import sys
    code = """
import importlib.util
real = importlib.util.spec_from_file_location
def missing(name, *args, **kwargs):
    if name == "_torch_layers":
        raise ImportError("no torch side")
    return real(name, *args, **kwargs)
importlib.util.spec_from_file_location = missing
import torch
from aimet_b200.v2 import nn as qnn
from aimet_b200.v2.quantsim import QuantizationSimModel
sim = QuantizationSimModel(torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.LayerNorm(4)))
for call in (lambda: qnn.linear(torch.zeros(2, 4), torch.zeros(3, 4)), lambda: qnn.layer_norm(torch.zeros(2, 4), 4)):
    try:
        call()
    except ImportError as e:
        assert "no torch side" in str(e)
    else:
        raise AssertionError("not refused")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


def test_torch_side_is_loaded_once():
    import threading
    from aimet_b200.v2 import nn as qnn
    found = []
    threads = [threading.Thread(target=lambda: found.append(qnn._layers)) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(found) == 8 and len({id(m) for m in found}) == 1 and callable(found[0].linear)
    with pytest.raises(AttributeError):
        qnn.no_such_name   # pylint: disable=pointless-statement


def test_torch_side_of_another_torch(monkeypatch, tmp_path):
    """The torch side is rebuilt for, and not loaded into, a torch or a Python other than the one it was built for."""
    import torch as installed
    from aimet_b200 import build
    from aimet_b200.v2 import nn as qnn
    commands = []

    def compiler(cmd, **_):
        commands.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w", encoding="utf-8") as f:
            f.write("library")
        return type("Done", (), {"returncode": 0, "stdout": "", "stderr": ""})()

    monkeypatch.setattr(build, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(build, "TORCH_PATH", str(tmp_path / "_torch_layers.so"))
    monkeypatch.setattr(build.subprocess, "run", compiler)
    build.build_torch()
    build.build_torch()
    assert len(commands) == 1 and not build.torch_side_is_foreign()
    monkeypatch.setattr(installed, "__version__", "9.9.9")
    assert build.torch_side_is_foreign()
    with pytest.raises(ImportError, match="another"):
        qnn._load()
    build.build_torch()
    assert len(commands) == 2 and not build.torch_side_is_foreign()


@pytest.mark.parametrize("bits", [10, 7])
def test_norm_bound_sees_operands_of_fewer_bits(bits):
    """The check of the float32 products fails for operands rounded to 10 bits (7: bfloat16) at every size it is used at."""
    from _layers import FLOAT32_SIZES, float32_norm_bound, norm_error
    g = torch.Generator().manual_seed(109)

    def cut(t):
        mantissa, exponent = torch.frexp(t)
        return torch.ldexp(torch.round(mantissa * 2 ** (bits + 1)) / 2 ** (bits + 1), exponent)

    for m, k, n in FLOAT32_SIZES:
        for depth, rows, cols in ((k, m, n), (n, m, k), (m, n, k)):
            a, b = (torch.randn(s, generator=g, dtype=torch.float32).double() for s in ((rows, depth), (depth, cols)))
            want = a @ b
            assert norm_error(cut(a) @ cut(b), want) > 4 * float32_norm_bound(depth)
            plain = (a.float() @ b.float()).double()
            assert norm_error(plain, want) <= float32_norm_bound(depth)


def test_fuse_layers_keeps_its_order_around_hooks(on_torch):
    """A hook of a module between the layer and its activation writes to the layer's input."""
    def hooked_between(s, x):
        h = x * 1.0
        y = s.a(h)
        g = s.i(h)
        return F.relu(y) * g

    torch.manual_seed(0)
    net = _Net(hooked_between, i=nn.Identity()).eval()

    def double(module, args):
        args[0].mul_(2.0)

    net.i.register_forward_pre_hook(double)
    x = torch.randn(5, 8)
    expect = net(x.clone())
    sim, _ = _fused(net)
    assert torch.allclose(sim.model(x.clone()), expect, atol=1e-6)
    assert on_torch == [("linear", None, False)]
