"""linear and layer_norm on the GPU against float64, forward and backward, over types, sizes, layouts and edge values."""
import copy

import pytest
import torch
from torch import nn
import torch.nn.functional as F

from _layers import ACTS, DTYPES, assert_within, act, linear_ref, norm_ref, slope

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)


def _check_linear(x, w, b, r, kind, dy, what=""):
    """Forward without gradients, then forward and backward, both against float64."""
    from aimet_b200.v2.nn import linear
    k, n = w.shape[1], w.shape[0]
    xm, rm = x.reshape(-1, k), None if r is None else r.reshape(-1, n)
    ref = linear_ref(xm, w, b, rm, kind, dy.reshape(-1, n))
    with torch.no_grad():
        y = linear(x, w, b, kind, r)
    assert y.shape == x.shape[:-1] + (n,) and y.dtype == x.dtype
    assert_within(y, ref["y"], what + " y")
    leaves = {name: t.detach().requires_grad_(True) for name, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None}
    y2 = linear(leaves["x"], leaves["w"], leaves.get("b"), kind, leaves.get("r"))
    assert torch.equal(y2.detach(), y), what + ": the result depends on whether gradients are wanted"
    grads = dict(zip(leaves, torch.autograd.grad(y2, list(leaves.values()), dy)))
    assert grads["x"].shape == x.shape
    assert_within(grads["x"], ref["dx"], what + " dx")
    assert_within(grads["w"], ref["dw"], what + " dw")
    if b is not None:
        assert_within(grads["b"], ref["db"], what + " db")
    if r is not None:
        assert torch.equal(grads["r"], dy)


LINEAR_SIZES = [
    # m, k, n
    (1, 1, 1), (1, 64, 8), (1, 4096, 512), (2, 7, 3), (5, 1000, 16), (8, 512, 1000), (9, 33, 65), (16, 256, 128),
    (17, 257, 129), (31, 2048, 333), (33, 40, 2000), (64, 64, 64), (65, 1001, 130), (100, 8, 72), (127, 129, 127),
    (128, 128, 128), (129, 192, 257), (200, 4000, 96), (255, 72, 520), (300, 520, 1), (257, 1, 260), (512, 768, 768),
    (1000, 65, 33), (1100, 600, 1544),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n", LINEAR_SIZES)
def test_linear_sizes(cuda, dtype, m, k, n):
    g = _gen(m * 1000003 + k * 1009 + n)
    kind = ACTS[(m + k + n) % 5]
    x, w = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype, scale=k ** -0.5)
    b = _randn(g, n, dtype=dtype) if (m + k) % 3 else None
    r = _randn(g, m, n, dtype=dtype) if (k + n) % 2 else None
    _check_linear(x, w, b, r, kind, _randn(g, m, n, dtype=dtype), f"{m}x{k}x{n} {kind}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m", [3, 150, 700])
def test_linear_epilogues(cuda, dtype, kind, bias, residual, m):
    g = _gen(7)
    k, n = 192, 264
    x, w = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype, scale=0.2)
    _check_linear(x, w, _randn(g, n, dtype=dtype) if bias else None, _randn(g, m, n, dtype=dtype) if residual else None,
                  kind, _randn(g, m, n, dtype=dtype), f"{kind}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m", [1, 6, 96, 600])
def test_linear_layouts(cuda, dtype, m):
    """Leading dimensions, column slices, odd starts, transposed storage, expanded rows, a strided gradient."""
    g = _gen(11)
    k, n = 136, 200
    w = _randn(g, n, k, dtype=dtype, scale=0.1)
    b = _randn(g, n, dtype=dtype)
    wide = _randn(g, m, k + 24, dtype=dtype)
    dyw = _randn(g, m, n + 1, dtype=dtype)
    for name, x in (("pitched", wide[:, 8:8 + k]), ("odd start", wide[:, 3:3 + k]),
                    ("columns", _randn(g, k, m, dtype=dtype).t()), ("one row repeated", wide[:1, :k].expand(m, k)),
                    ("every other", _randn(g, m, 2 * k, dtype=dtype)[:, ::2]), ("reversed pitch", wide.flip(0)[:, :k])):
        _check_linear(x, w, b, None, "gelu", dyw[:, 1:], name)
    _check_linear(_randn(g, 2, 3, m, k, dtype=dtype).transpose(0, 2), w, b, _randn(g, m, 3, 2, n, dtype=dtype), "silu",
                  _randn(g, m, 3, 2, n, dtype=dtype), "four dimensions")
    x = wide[:, :k]
    for name, w2 in (("transposed weight", _randn(g, k, n, dtype=dtype, scale=0.1).t()),
                     ("odd weight", _randn(g, n, k + 5, dtype=dtype, scale=0.1)[:, 5:])):
        _check_linear(x, w2, _randn(g, 2 * n, dtype=dtype)[::2], _randn(g, m, 2 * n, dtype=dtype)[:, ::2], "relu",
                      _randn(g, 1, n, dtype=dtype).expand(m, n), name)
    from aimet_b200.v2.nn import linear
    row = _randn(g, k, dtype=dtype)
    assert torch.equal(linear(row, w, b), linear(row[None], w, b)[0])


def test_linear_one_million_rows(cuda):
    """More rows than a grid dimension has blocks, and more than 2^31 bytes of output."""
    g = _gen(13)
    m, k, n = (1 << 20) + 5, 16, 1040
    x, w = _randn(g, m, k, dtype=torch.bfloat16), _randn(g, n, k, dtype=torch.bfloat16)
    from aimet_b200.v2.nn import linear
    with torch.no_grad():
        y = linear(x, w)
    rows = torch.tensor([0, 1, 65535, 65536, 524287, 1032443, 1048576, m - 1], device="cuda")
    assert_within(y[rows], linear_ref(x[rows], w, None, None, None)["y"], "rows")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_linear_empty(cuda, dtype):
    from aimet_b200.v2.nn import linear
    x = torch.empty(0, 24, device=cuda, dtype=dtype, requires_grad=True)
    w = torch.ones(8, 24, device=cuda, dtype=dtype, requires_grad=True)
    b = torch.ones(8, device=cuda, dtype=dtype, requires_grad=True)
    y = linear(x, w, b, "gelu", torch.empty(0, 8, device=cuda, dtype=dtype))
    assert y.shape == (0, 8)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert dx.shape == (0, 24) and not dw.any() and not db.any() and dw.shape == (8, 24)
    assert linear(x.detach().reshape(3, 0, 24), w, b).shape == (3, 0, 8)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(4, 80, 96), (300, 264, 272), (140, 65, 33)])
def test_linear_inf_and_nan_stay_in_their_rows(cuda, dtype, m, k, n):
    """A row with infinities or NaN changes its own results and no other row's."""
    from aimet_b200.v2.nn import linear
    g = _gen(17)
    x, w = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype)
    w[w == 0] = 1
    clean = linear(x, w, None, "relu")
    bad = x.clone()
    bad[1, 3], bad[m - 1, k - 1] = float("nan"), float("inf")
    y = linear(bad, w, None, "relu")
    assert torch.equal(y[2:m - 1], clean[2:m - 1]) and torch.equal(y[0], clean[0])
    assert bool(y[1].isnan().all())
    assert bool(torch.where(w[:, k - 1] > 0, y[m - 1] == float("inf"), y[m - 1] == 0).all())


@pytest.mark.parametrize("kind", ACTS[1:])
def test_activation_limits(cuda, kind):
    """Large arguments: values and slopes take their limits, nothing overflows on the way."""
    from aimet_b200.v2.nn import linear
    z = torch.tensor([-1e30, -3e4, -200., -50., -14.5, -13., -5., -1e-3, -0., 0., 1e-3, 5., 13., 14.5, 50., 200., 3e4, 1e30],
                     device=cuda)
    x = z[:, None].clone().requires_grad_(True)
    y = linear(x, torch.ones(1, 1, device=cuda), None, kind)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    zz = z.double().requires_grad_(True)
    want = F.relu(zz) if kind == "relu" else F.silu(zz) if kind == "silu" else \
        F.gelu(zz, approximate="tanh" if kind == "gelu_tanh" else "none")
    (slope,) = torch.autograd.grad(want.sum(), zz)
    slope = torch.nan_to_num(slope, nan=1.0)   # the formula's 0 * inf at 1e30
    torch.testing.assert_close(y[:, 0].double(), want.detach(), rtol=1e-5, atol=2e-6)
    torch.testing.assert_close(dx[:, 0].double(), slope, rtol=1e-5, atol=2e-6)


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=str)
@pytest.mark.parametrize("kind", ACTS[1:])
@pytest.mark.parametrize("m,n", [(1, 40), (20, 40), (300, 264), (300, 265)])
def test_activation_limits_in_16_bits(cuda, kind, dtype, m, n):
    """The same in the epilogues of the matrix products and in their backward pass, and NaN stays NaN."""
    from aimet_b200.v2.nn import linear
    z = torch.tensor([-6e4, -3e3, -200., -50., -14.5, -13.5, -5., -0.5, -1e-3, 0., 1e-3, 0.5, 5., 13.5, 14.5, 50., 200., 6e4],
                     device=cuda).to(dtype)
    x = torch.zeros(m, 64, device=cuda, dtype=dtype)
    w = torch.zeros(n, 64, device=cuda, dtype=dtype)
    x[:, 3] = 1
    w[:, 3] = z.repeat(n)[:n]
    x.requires_grad_(True)
    b = torch.zeros(n, device=cuda, dtype=dtype, requires_grad=True)
    y = linear(x, w, b, kind)
    (db,) = torch.autograd.grad(y, b, torch.cat([torch.ones(1, n, device=cuda), torch.zeros(m - 1, n, device=cuda)]).to(dtype))
    zz = w[:, 3].double()
    half = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    # one rounding to the type; the functions themselves are good to 16 steps of 2^-24 of max(1, |z|)
    want, steep = act(zz, kind), slope(zz, kind)
    err = (y[0].double() - want).abs()
    assert bool((err <= half * want.abs() + 16 * 2.0 ** -24 * zz.abs().clamp_min(1)).all())
    assert bool(((db.double() - steep).abs() <= half * steep.abs() + 32 * 2.0 ** -24).all())
    bad = x.detach().clone()
    bad[0, 5] = float("nan")
    out = linear(bad, w, b.detach(), kind)
    assert bool(out[0].isnan().all()) and not bool(out[1:].isnan().any())


@pytest.mark.parametrize("kind", ACTS)
def test_linear_gradients_against_differences(cuda, kind):
    """Directional derivatives of a float64 loss by central differences."""
    from aimet_b200.v2.nn import linear
    g = _gen(19)
    m, k, n = 37, 52, 44
    p = {"x": _randn(g, m, k), "w": _randn(g, n, k, scale=0.2), "b": _randn(g, n), "r": _randn(g, m, n)}
    dy = _randn(g, m, n)
    leaves = {a: t.clone().requires_grad_(True) for a, t in p.items()}
    y = linear(leaves["x"], leaves["w"], leaves["b"], kind, leaves["r"])
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))

    def loss(q):
        return ((act(q["x"] @ q["w"].t() + q["b"], kind) + q["r"]) * dy.double()).sum()

    base = {a: t.double() for a, t in p.items()}
    for a in p:
        d = _randn(g, *p[a].shape).double()
        h = 1e-6
        num = (loss({**base, a: base[a] + h * d}) - loss({**base, a: base[a] - h * d})) / (2 * h)
        ana = (grads[a].double() * d).sum()
        scale = (grads[a].double().abs() * d.abs()).sum()
        # float32 sums: (n + 8) steps of 2^-23; the difference itself: h^2 and 1e-16 / h; a corner of relu may be crossed
        assert abs(float(num - ana)) <= 1e-4 * float(scale), (a, float(num), float(ana))


def test_linear_only_some_gradients(cuda):
    from aimet_b200.v2.nn import linear
    g = _gen(23)
    p = {"x": _randn(g, 70, 48), "w": _randn(g, 40, 48), "b": _randn(g, 40), "r": _randn(g, 70, 40)}
    dy = _randn(g, 70, 40)
    for kind in (None, "silu"):
        full = {a: t.clone().requires_grad_(True) for a, t in p.items()}
        want = dict(zip(p, torch.autograd.grad(linear(full["x"], full["w"], full["b"], kind, full["r"]),
                                               list(full.values()), dy)))
        for a in p:
            one = {c: t.clone().requires_grad_(c == a) for c, t in p.items()}
            (got,) = torch.autograd.grad(linear(one["x"], one["w"], one["b"], kind, one["r"]), one[a], dy)
            assert torch.equal(got, want[a]), (kind, a)


def test_linear_same_tensor_twice(cuda):
    """x as its own weight and residual: the gradients of all three uses add up."""
    from aimet_b200.v2.nn import linear
    g = _gen(29)
    x = _randn(g, 96, 96, scale=0.1).requires_grad_(True)
    dy = _randn(g, 96, 96)
    (got,) = torch.autograd.grad(linear(x, x, None, "silu", x), x, dy)
    xd = x.detach().double().requires_grad_(True)
    (want,) = torch.autograd.grad(F.silu(xd @ xd.t()) + xd, xd, dy.double())
    torch.testing.assert_close(got.double(), want, rtol=1e-4, atol=1e-4)


def test_linear_in_place_change_is_noticed(cuda):
    from aimet_b200.v2.nn import linear
    x = torch.randn(16, 16, device=cuda)
    w = torch.randn(16, 16, device=cuda, requires_grad=True)
    y = linear(x, w)
    x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_linear_repeats_bit_for_bit(cuda, dtype):
    from aimet_b200.v2.nn import linear
    g = _gen(31)
    for m, k, n in ((1, 4096, 1032), (24, 2048, 520), (300, 1024, 136), (2049, 264, 264)):
        x, w = _randn(g, m, k, dtype=dtype).requires_grad_(True), _randn(g, n, k, dtype=dtype).requires_grad_(True)
        b = _randn(g, n, dtype=dtype).requires_grad_(True)
        dy = _randn(g, m, n, dtype=dtype)
        first = None
        for _ in range(4):
            y = linear(x, w, b, "gelu")
            now = [y.detach(), *torch.autograd.grad(y, [x, w, b], dy)]
            if first is None:
                first = now
            assert all(torch.equal(p, q) for p, q in zip(first, now))


def test_linear_leaves_its_surroundings_alone(cuda):
    """Results land in freshly allocated memory; what lies around operands and results keeps its bits."""
    from aimet_b200._lib import check, lib

    def forward(x, w, y, z=None):
        code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[x.dtype]
        check(lib.aq_linear_forward(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), None, None, 0, y.data_ptr(), y.stride(0),
                                    None if z is None else z.data_ptr(), 0 if z is None else z.stride(0), code, x.shape[0],
                                    w.shape[0], x.shape[1], 1, torch.cuda.current_stream().cuda_stream))

    for dtype in DTYPES:
        for m, k, n in ((3, 72, 40), (130, 136, 264), (513, 64, 520)):
            g = _gen(37)
            x, w = _randn(g, m, k, dtype=dtype), _randn(g, n, k, dtype=dtype)
            big = torch.full((m + 4, n + 16), 7.0, device=cuda, dtype=dtype)
            zbig = torch.full((m + 4, n + 16), 7.0, device=cuda, dtype=dtype)
            forward(x, w, big[2:2 + m, 8:8 + n], zbig[2:2 + m, 8:8 + n])
            for t in (big, zbig):
                edge = t.clone()
                edge[2:2 + m, 8:8 + n] = 7.0
                assert bool((edge == 7.0).all()), (dtype, m, k, n)
            ref = linear_ref(x, w, None, None, "relu")["y"]
            assert_within(big[2:2 + m, 8:8 + n], ref, "pitched result")
            big = torch.full((m + 4, n + 15), 7.0, device=cuda, dtype=dtype)   # odd pitch, odd start
            forward(x, w, big[2:2 + m, 7:7 + n])
            assert_within(big[2:2 + m, 7:7 + n], ref, "odd result")
            big[2:2 + m, 7:7 + n] = 7.0
            assert bool((big == 7.0).all()), (dtype, m, k, n)


# ---- layer norm --------------------------------------------------------------------------------------------------
def _check_norm(x, shape, w, b, eps, dy, what=""):
    from aimet_b200.v2.nn import layer_norm
    dim = 1
    for s in shape:
        dim *= s
    ref = norm_ref(x.reshape(-1, dim), w, b, eps, dy.reshape(-1, dim))
    with torch.no_grad():
        y = layer_norm(x, shape, w, b, eps)
    assert y.shape == x.shape and y.dtype == x.dtype
    assert_within(y, ref["y"], what + " y")
    leaves = {n: t.detach().requires_grad_(True) for n, t in (("x", x), ("w", w), ("b", b)) if t is not None}
    y2 = layer_norm(leaves["x"], shape, leaves.get("w"), leaves.get("b"), eps)
    assert torch.equal(y, y2.detach())
    grads = dict(zip(leaves, torch.autograd.grad(y2, list(leaves.values()), dy)))
    for n in grads:
        assert grads[n].shape == leaves[n].shape
        assert_within(grads[n], ref["d" + n], f"{what} d{n}")


NORM_SIZES = [(1, 1), (1, 8), (3, 5), (1, 4096), (7, 64), (33, 100), (2, 1000), (65, 127), (9, 1537), (5, 2048), (300, 768),
              (4, 8191), (3, 11008), (2, 16384), (2, 16391), (1, 40000), (2, 70000), (1500, 24), (1025, 260), (4097, 9)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,dim", NORM_SIZES)
def test_norm_sizes(cuda, dtype, rows, dim):
    g = _gen(rows * 7919 + dim)
    x = _randn(g, rows, dim, dtype=dtype, shift=0.5)
    w = _randn(g, dim, dtype=dtype, scale=0.2, shift=1.0) if (rows + dim) % 4 else None
    b = _randn(g, dim, dtype=dtype, scale=0.2) if dim % 3 else None
    _check_norm(x, (dim,), w, b, 1e-5, _randn(g, rows, dim, dtype=dtype), f"{rows}x{dim}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dim", [40, 1024, 4104])
def test_norm_layouts(cuda, dtype, dim):
    g = _gen(41)
    rows = 37
    w, b = _randn(g, dim, dtype=dtype, shift=1.0), _randn(g, dim, dtype=dtype)
    wide = _randn(g, rows, dim + 24, dtype=dtype, scale=3.0, shift=-1.0)
    dy = _randn(g, rows, dim, dtype=dtype)
    for name, x in (("pitched", wide[:, 16:16 + dim]), ("odd start", wide[:, 3:3 + dim]),
                    ("columns", _randn(g, dim, rows, dtype=dtype).t()), ("one row repeated", wide[:1, :dim].expand(rows, dim))):
        _check_norm(x, (dim,), w, b, 1e-5, dy, name)
    _check_norm(wide[:, :dim], (dim,), _randn(g, 2 * dim, dtype=dtype)[::2], _randn(g, dim + 1, dtype=dtype)[1:], 1e-5,
                _randn(g, rows, dim + 3, dtype=dtype)[:, 3:], "odd weight, odd gradient")
    _check_norm(wide[:, :dim], (dim,), w, b, 1e-5, _randn(g, 1, dim, dtype=dtype).expand(rows, dim), "one gradient row")
    shape = (4, dim // 4)
    _check_norm(_randn(g, 5, 6, *shape, dtype=dtype).transpose(0, 1), shape, w.reshape(shape), b.reshape(shape), 1e-3,
                _randn(g, 6, 5, *shape, dtype=dtype), "two normalised dimensions")
    from aimet_b200.v2.nn import layer_norm
    assert torch.equal(layer_norm(wide[0, :dim], dim, w, b), layer_norm(wide[:1, :dim], dim, w, b)[0])
    bias_only = b.reshape(shape).clone().requires_grad_(True)
    layer_norm(wide[:, :dim].reshape(rows, *shape), shape, None, bias_only).float().sum().backward()
    assert bias_only.grad.shape == shape


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dim", [65, 300, 512, 513, 519, 777, 1001, 1537, 2051, 4096, 4099, 5001, 6145, 8193, 12001, 16391, 20001])
def test_norm_rows_off_boundaries(cuda, dtype, dim):
    """Many rows of odd lengths and pitches, each tensor with its own alignment; what lies between the rows is NaN."""
    g = _gen(61 + dim)
    rows = 745 + dim % 5

    def inside(start, pad, **kw):
        wide = torch.full((rows, dim + start + pad), float("nan"), device=cuda, dtype=dtype)
        wide[:, start:start + dim] = _randn(g, rows, dim, dtype=dtype, **kw)
        return wide[:, start:start + dim]

    w, b = _randn(g, dim + 1, dtype=dtype, shift=1.0)[1:], _randn(g, dim + 3, dtype=dtype)[3:]
    for k, (x, dy) in enumerate(((inside(0, 0, shift=0.5), inside(0, 0)), (inside(3, 0), inside(0, 1)),
                                 (inside(1, 8), inside(8, 7)))):
        _check_norm(x, (dim,), w if k != 1 else None, b if k != 2 else None, 1e-5, dy, f"{rows}x{dim} layout {k}")
    from aimet_b200.v2.nn import layer_norm
    x, dy = inside(5, 2).requires_grad_(True), inside(0, 3)
    ref = norm_ref(x, w, b, 1e-5, dy)
    for name, leaf, args in (("dx", x, (x, w, b)), ("dw", w.requires_grad_(True), (x.detach(), w, b)),
                             ("db", b.requires_grad_(True), (x.detach(), w.detach(), b))):
        y = layer_norm(args[0], dim, args[1], args[2], 1e-5)
        assert_within(torch.autograd.grad(y, leaf, dy)[0], ref[name], name + " alone")


@pytest.mark.parametrize("dtype", DTYPES[::2], ids=str)
@pytest.mark.parametrize("rows,dim", [(5, 40), (5, 65), (5, 1000), (800, 40), (800, 65), (800, 1000), (800, 1001)])
def test_norm_large_constant_rows(cuda, dtype, rows, dim):
    """mean rstd passes float32's range, h does not: 2^117 and its sums over a row are exact, so h is 0 and
    dx = rstd (dy - mean dy)."""
    from aimet_b200.v2.nn import layer_norm
    g = _gen(67)
    x = torch.full((rows, dim), 2.0 ** 117, device=cuda, dtype=dtype, requires_grad=True)
    dy = _randn(g, rows, dim, dtype=dtype)
    y = layer_norm(x, dim, None, None, 1e-12)
    assert not bool(y.detach().any())
    (dx,) = torch.autograd.grad(y, x, dy)
    d = dy.double()
    mean, size = d.mean(1, keepdim=True), d.abs().mean(1, keepdim=True)
    want = 1e6 * (d - mean)
    # the sum of dim terms and its quotient; the products with rstd and the difference; rstd's root and quotient; the result
    e = 1e6 * ((dim + 8) * 2.0 ** -24 * size + 3 * 2.0 ** -24 * (d.abs() + size)) + 4 * 2.0 ** -24 * want.abs()
    u = torch.finfo(dtype).eps / 2
    assert bool(((dx.double() - want).abs() <= e * (1 + u) + u * want.abs()).all())


@pytest.mark.parametrize("dim", [96, 1024, 1537, 11008, 40000])
def test_norm_mean_far_from_zero(cuda, dim):
    """|mean| a thousand times the spread: the variance is not formed as a difference of two large numbers."""
    g = _gen(43)
    x = _randn(g, 6, dim, shift=1000.0)
    _check_norm(x, (dim,), None, None, 1e-5, _randn(g, 6, dim), "far mean")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dim", [1, 64, 4096, 40000])
def test_norm_constant_rows(cuda, dtype, dim):
    """A spread of zero: y is the bias, and dx is what eps leaves."""
    from aimet_b200.v2.nn import layer_norm
    x = torch.full((3, dim), 2.0, device=cuda, dtype=dtype, requires_grad=True)
    b = torch.randn(dim, device=cuda).to(dtype)
    y = layer_norm(x, dim, None, b, 1e-5)
    assert torch.equal(y.detach(), b.expand(3, dim))
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert bool((dx == 0).all())


@pytest.mark.parametrize("rows,dim", [(40, 64), (40, 1000), (40, 4096), (40, 40000), (800, 65), (800, 1001), (800, 4101)])
def test_norm_inf_and_nan_stay_in_their_rows(cuda, rows, dim):
    from aimet_b200.v2.nn import layer_norm
    g = _gen(47)
    x = _randn(g, rows, dim, dtype=torch.bfloat16)
    clean = layer_norm(x, dim)
    bad = x.clone()
    bad[3, 5], bad[17, dim - 1] = float("nan"), float("inf")
    y = layer_norm(bad, dim)
    keep = [i for i in range(rows) if i not in (3, 17)]
    assert torch.equal(y[keep], clean[keep]) and bool(y[3].isnan().all()) and bool(y[17].isnan().all())
    bad.requires_grad_(True)
    dy = _randn(g, rows, dim, dtype=torch.bfloat16)
    (dx,) = torch.autograd.grad(layer_norm(bad, dim), bad, dy)
    assert bool(dx[keep].isfinite().all()) and not bool(dx[[3, 17]].isfinite().any())


def test_norm_empty(cuda):
    from aimet_b200.v2.nn import layer_norm
    x = torch.empty(0, 32, device=cuda, requires_grad=True)
    w = torch.ones(32, device=cuda, requires_grad=True)
    b = torch.ones(32, device=cuda, requires_grad=True)
    y = layer_norm(x, 32, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert y.shape == (0, 32) and dx.shape == (0, 32) and not dw.any() and not db.any()


def test_norm_many_rows(cuda):
    """More rows than a grid dimension has blocks; the parameter gradients' sums over all of them."""
    g = _gen(53)
    _check_norm(_randn(g, 200001, 16, dtype=torch.float16), (16,), _randn(g, 16, dtype=torch.float16),
                _randn(g, 16, dtype=torch.float16), 1e-5, _randn(g, 200001, 16, dtype=torch.float16, scale=0.01), "many rows")


@pytest.mark.parametrize("dim", [48, 1536, 20000])
def test_norm_gradients_against_differences(cuda, dim):
    from aimet_b200.v2.nn import layer_norm
    g = _gen(59)
    p = {"x": _randn(g, 9, dim), "w": _randn(g, dim, shift=1.0), "b": _randn(g, dim)}
    dy = _randn(g, 9, dim)
    leaves = {a: t.clone().requires_grad_(True) for a, t in p.items()}
    grads = dict(zip(p, torch.autograd.grad(layer_norm(leaves["x"], dim, leaves["w"], leaves["b"]), list(leaves.values()), dy)))
    base = {a: t.double() for a, t in p.items()}

    def loss(q):
        return (F.layer_norm(q["x"], (dim,), q["w"], q["b"], 1e-5) * dy.double()).sum()

    for a in p:
        d = _randn(g, *p[a].shape).double()
        h = 1e-5
        num = (loss({**base, a: base[a] + h * d}) - loss({**base, a: base[a] - h * d})) / (2 * h)
        ana = (grads[a].double() * d).sum()
        assert abs(float(num - ana)) <= 1e-5 * float((grads[a].double().abs() * d.abs()).sum()), a


def test_norm_some_gradients_and_bits(cuda):
    from aimet_b200.v2.nn import layer_norm
    g = _gen(61)
    for rows, dim in ((300, 264), (40, 4096), (17, 1537), (3, 40000)):
        p = {"x": _randn(g, rows, dim), "w": _randn(g, dim), "b": _randn(g, dim)}
        dy = _randn(g, rows, dim)
        full = {a: t.clone().requires_grad_(True) for a, t in p.items()}
        want = dict(zip(p, torch.autograd.grad(layer_norm(full["x"], dim, full["w"], full["b"]), list(full.values()), dy)))
        for a in p:
            one = {c: t.clone().requires_grad_(c == a) for c, t in p.items()}
            (got,) = torch.autograd.grad(layer_norm(one["x"], dim, one["w"], one["b"]), one[a], dy)
            assert torch.equal(got, want[a]), (rows, dim, a)


# ---- streams, graphs, several calls at once ------------------------------------------------------------------------
def _block(p, x):
    from aimet_b200.v2.nn import layer_norm, linear
    h = layer_norm(x, x.shape[-1], p["nw"], p["nb"])
    h = linear(h, p["w1"], p["b1"], "gelu")
    return linear(h, p["w2"], p["b2"], None, x)


def _block_params(g, d, f, dtype):
    return {"nw": _randn(g, d, dtype=dtype, scale=0.1, shift=1.0), "nb": _randn(g, d, dtype=dtype, scale=0.1),
            "w1": _randn(g, f, d, dtype=dtype, scale=d ** -0.5), "b1": _randn(g, f, dtype=dtype, scale=0.1),
            "w2": _randn(g, d, f, dtype=dtype, scale=f ** -0.5), "b2": _randn(g, d, dtype=dtype, scale=0.1)}


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,d,f", [(1, 256, 1024), (50, 136, 520), (700, 512, 1408)])
def test_block_together(cuda, dtype, rows, d, f):
    """Norm, up projection with gelu, down projection onto the residual stream: forward and every gradient."""
    g = _gen(67)
    p = {a: t.requires_grad_(True) for a, t in _block_params(g, d, f, dtype).items()}
    x = _randn(g, rows, d, dtype=dtype).requires_grad_(True)
    dy = _randn(g, rows, d, dtype=dtype)
    y = _block(p, x)
    got = [y.detach(), *torch.autograd.grad(y, [x, *p.values()], dy)]
    q = {a: t.detach().double().requires_grad_(True) for a, t in p.items()}
    xd = x.detach().double().requires_grad_(True)
    h = F.layer_norm(xd, (d,), q["nw"], q["nb"], 1e-5)
    yd = F.linear(F.gelu(F.linear(h, q["w1"], q["b1"])), q["w2"], q["b2"]) + xd
    want = [yd.detach(), *torch.autograd.grad(yd, [xd, *q.values()], dy.double())]
    # each of the six roundings to the storage type between input and result moves a value by at most half a step of
    # its size, and random signs average over the sums: 8 half steps of the tensor's norm cover them in every tensor
    half = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    tol = 8 * half if dtype != torch.float32 else 64 * half   # float32: the sums' own rounding over up to 1408 terms
    for a, b in zip(got, want):
        assert float((a.double() - b).norm()) <= tol * float(b.norm())


def test_side_stream_and_graph_replay(cuda):
    """A captured forward and backward pass, replayed with new inputs, equals the eager passes bit for bit."""
    g = _gen(71)
    dtype = torch.bfloat16
    for rows in (1, 24, 300):
        p = {a: t.requires_grad_(True) for a, t in _block_params(g, 264, 1032, dtype).items()}
        xs = [_randn(g, rows, 264, dtype=dtype) for _ in range(3)]
        dy = _randn(g, rows, 264, dtype=dtype)
        x = xs[0].clone().requires_grad_(True)

        def step():
            y = _block(p, x)
            return [y.detach(), *torch.autograd.grad(y, [x, *p.values()], dy)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for v in xs:
            with torch.no_grad():
                x.copy_(v)
            graph.replay()
            replayed = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(replayed, step()))


def test_two_streams_at_once(cuda):
    """Calls on two streams, and two captured graphs replayed side by side, do not share scratch memory."""
    g = _gen(73)
    dtype = torch.float16
    jobs = []
    for rows, d, f in ((40, 2056, 520), (600, 264, 776)):
        p = {a: t.requires_grad_(True) for a, t in _block_params(g, d, f, dtype).items()}
        x = _randn(g, rows, d, dtype=dtype).requires_grad_(True)
        dy = _randn(g, rows, d, dtype=dtype)

        def step(p=p, x=x, dy=dy):
            y = _block(p, x)
            return [y.detach(), *torch.autograd.grad(y, [x, *p.values()], dy)]
        jobs.append(step)
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(10):
        for i, (job, s) in enumerate(zip(jobs, streams)):
            with torch.cuda.stream(s):
                got[i].append(job())
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(res, want[i]))
    graphs, outs = [], []
    for job in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(job())
        graphs.append(graph)
    for _ in range(10):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))


def test_quantized_tensors_count_as_numbers(cuda):
    """Fake-quantized tensors that carry their encoding: same numbers, plain result, gradients through the quantizer."""
    from aimet_b200.v2.nn import layer_norm, linear
    from aimet_b200.v2.quantizer import QuantizeDequantize
    g = _gen(79)
    w = _randn(g, 40, 64).requires_grad_(True)
    q = QuantizeDequantize((40, 1), 8, True).to(cuda)
    with q.compute_encodings():
        q(w)
    wq = q(w)
    assert type(wq) is not torch.Tensor
    x = _randn(g, 30, 64)
    y = linear(x, wq, None, "relu")
    assert type(y) is torch.Tensor and torch.equal(y, linear(x, wq.detach().as_subclass(torch.Tensor), None, "relu"))
    (dw,) = torch.autograd.grad(y.sum(), w)
    assert dw.shape == w.shape and bool(dw.any())
    assert type(layer_norm(wq, 64)) is torch.Tensor


def test_inference_mode_and_backward_accumulation(cuda):
    from aimet_b200.v2.nn import layer_norm, linear
    g = _gen(83)
    x, w = _randn(g, 20, 32), _randn(g, 24, 32).requires_grad_(True)
    with torch.inference_mode():
        y = linear(layer_norm(x, 32), w)
    assert not y.requires_grad
    for _ in range(2):   # gradients add up in the leaf
        linear(x, w).sum().backward()
    torch.testing.assert_close(w.grad, 2 * x.sum(0).expand(24, 32), rtol=1e-5, atol=1e-5)


def test_refusals_on_the_gpu(cuda):
    from aimet_b200._lib import lib
    from aimet_b200.v2.nn import layer_norm, linear
    x, w = torch.randn(4, 16, device=cuda), torch.randn(8, 16, device=cuda)
    with pytest.raises(RuntimeError, match="weight is"):
        linear(x, w.half())
    with pytest.raises(RuntimeError, match="residual must have shape"):
        linear(x, w, residual=torch.zeros(8, device=cuda))
    with pytest.raises(RuntimeError, match="bias must have shape"):
        linear(x, w, torch.zeros(4, device=cuda))
    with pytest.raises(RuntimeError, match="cannot apply"):
        linear(x[:, :15], w)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        linear(x, w.cpu())
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        linear(x.double(), w.double())
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="tanh")
    with pytest.raises(RuntimeError, match="cannot normalise"):
        layer_norm(x, 8)
    with pytest.raises(RuntimeError, match="weight must have shape"):
        layer_norm(x, 16, w)
    with pytest.raises(RuntimeError, match="eps"):
        layer_norm(x, 16, eps=-1.0)
    xr = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(linear(xr, w, None, "silu").sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        dx.sum().backward()
    # the C entry refuses rows the tensor cores cannot read
    h = torch.zeros(12, 24, device=cuda, dtype=torch.float16)
    y = torch.zeros(12, 4, device=cuda, dtype=torch.float16)
    assert lib.aq_linear_forward(h.data_ptr() + 2, 24, h.data_ptr(), 24, None, None, 0, y.data_ptr(), 4, None, 0, 1, 9, 4, 8,
                                 0, None) == -1
    assert lib.aq_linear_forward(h.data_ptr(), 23, h.data_ptr(), 24, None, None, 0, y.data_ptr(), 4, None, 0, 1, 9, 4, 8,
                                 0, None) == -1


# ---- through the simulated model -----------------------------------------------------------------------------------
class _Mlp(nn.Module):
    def __init__(self, d=64, f=160):
        super().__init__()
        self.norm, self.up, self.act, self.down = nn.LayerNorm(d), nn.Linear(d, f), nn.GELU(), nn.Linear(f, d)
        self.gate, self.relu = nn.Linear(d, f), nn.ReLU()

    def forward(self, x):
        h = self.norm(x)
        return self.down(self.act(self.up(h)) + self.relu(self.gate(h))) + x


@pytest.mark.parametrize("without_activation_quantizers", [False, True])
def test_quantsim_fused_layers(cuda, without_activation_quantizers):
    """The simulated model gives the same results on the kernels as on torch's layers, and trains the same way."""
    from aimet_b200.v2.quantsim import QuantizationSimModel
    torch.manual_seed(3)
    model = _Mlp().to(cuda)
    data = [torch.randn(33, 64, device=cuda) for _ in range(2)]
    sim = QuantizationSimModel(model, data[0], quant_scheme="post_training_tf", default_output_bw=16)
    sim.compute_encodings(lambda m, _: [m(x) for x in data])
    if without_activation_quantizers:
        enc = sim.get_encodings_dict()
        sim.load_encodings({"param_encodings": enc["param_encodings"], "activation_encodings": {}}, partial=False)
    fused = copy.deepcopy(sim)
    assert fused.fuse_layers() > 0
    assert [type(m).__name__ for m in fused.layers.values()] == ["QuantizedLinear"] * 3
    if without_activation_quantizers:
        assert fused.get_encodings_dict() == sim.get_encodings_dict()
    x = data[0]
    out = []
    for s in (sim, fused):
        y = s.model(x)
        y.square().mean().backward()
        out.append((y.detach(), [l.layer.weight.grad for l in s.layers.values()], s.model.norm.weight.grad))
    # a 16-bit activation quantizer may move a value by one step of its range / 65535 where the two sums straddle a border
    step = max(float(q.get_scale().max()) for q in sim.activation_quantizers.values()) if sim.activation_quantizers else 0.0
    torch.testing.assert_close(out[0][0], out[1][0], rtol=1e-4, atol=1e-4 + 4 * step)
    for a, b in zip(out[0][1] + [out[0][2]], out[1][1] + [out[1][2]]):
        assert float((a - b).norm()) <= 2e-3 * float(a.norm())


def test_no_wait_ran_out(cuda):
    """Runs last in this file: none of the products above gave up on a wait."""
    import ctypes
    from aimet_b200._lib import lib
    out = ctypes.c_int(7)
    assert lib.aq_layers_stuck(ctypes.byref(out)) == 0 and out.value == 0
