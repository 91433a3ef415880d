"""What linear and layer_norm do not differentiate they refuse."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 20])
def test_forward_mode_is_refused(cuda, m):
    from aimet_b200.v2.nn import layer_norm, linear
    x, w = torch.randn(m, 32, device=cuda), torch.randn(24, 32, device=cuda)
    for needs_grad in (False, True):
        w.requires_grad_(needs_grad)
        with fwad.dual_level():
            dx = fwad.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match="forward-mode"):
                linear(dx, w)
            with pytest.raises(RuntimeError, match="forward-mode"):
                layer_norm(dx, 32)
    xr = x.clone().requires_grad_(True)
    for y in (linear(xr, w.detach(), activation="gelu"), layer_norm(xr, 32)):
        with fwad.dual_level():
            dy = fwad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, xr, dy)


def test_function_transforms_are_refused(cuda):
    """Tensors that torch.func wraps have no memory of their own."""
    from aimet_b200.v2.nn import layer_norm, linear
    x, w = torch.randn(6, 5, 32, device=cuda), torch.randn(24, 32, device=cuda)
    for fn in (lambda t: linear(t, w), lambda t: layer_norm(t, 32)):
        with pytest.raises(RuntimeError):
            torch.func.vmap(fn)(x)
        with pytest.raises(RuntimeError):
            torch.func.jvp(fn, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t, fn=fn: fn(t).sum())(x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 20])
def test_lazily_negated_tensors(cuda, dtype, m):
    """Operands, parameters and gradients whose memory holds the negated values."""
    from aimet_b200.v2.nn import layer_norm, linear
    g = torch.Generator(device="cuda").manual_seed(103)
    x, w, b, r, dy, u, v = (torch.randn(s, device=cuda, generator=g).to(dtype)
                            for s in ((m, 32), (24, 32), (24,), (m, 24), (m, 24), (32,), (32,)))
    lazy = lambda t: torch._neg_view(t.neg())   # noqa: E731  (the same numbers)
    assert lazy(x).is_neg()
    assert torch.equal(linear(lazy(x), lazy(w), lazy(b), "gelu", lazy(r)), linear(x, w, b, "gelu", r))
    assert torch.equal(layer_norm(lazy(x), 32, lazy(u), lazy(v)), layer_norm(x, 32, u, v))
    leaves = [t.requires_grad_(True) for t in (x, w, b, u, v)]
    y = linear(layer_norm(x, 32, u, v), w, b, "silu")
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    got = torch.autograd.grad(y, leaves, lazy(dy))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
