"""Layer norm kernels against the formula in 64 bits (B200).

Tolerances, derived before the first run.  u = 2^-24.  The mean of d values is off by at most a few u of
the row's largest |x|, so x - mu is off by about (1 + few) u max|x|, xhat by that times rstd plus a few u
|xhat|: with A = max|x| rstd of the row, |err xhat| <= 16 u (A + |xhat|).  y adds one product and one sum:
<= 16 u ((A + |xhat|) |w| + |b|).  dx is rstd times three terms of size max|g| (A errors enter through
xhat): <= 64 u rstd (1 + A) max|g| (1 + max|xhat|).  dw and db are sums of N products in fp32, in chains no longer than
N/8: <= 2 u sqrt(N) ... bounded here by 8 u sqrt(N) times the root of the sum of squares, plus xhat's error.
A result of 16 bits adds half an ulp: 2^-8 (bf16, 8 significant bits) or 2^-11 (fp16, with 2^-25 below its normal range) of the value.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _layer_norm(*a, **k):
    from tensor_train_ing_b200.ops.layer_norm import layer_norm
    return layer_norm(*a, **k)


def _inputs(n, d, dtype, out, seed=0, bias=True, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(n, d, device="cuda", generator=g) * 1.5 + shift).to(dtype)
    w = 1 + 0.3 * torch.randn(d, device="cuda", generator=g)
    b = 0.2 * torch.randn(d, device="cuda", generator=g) if bias else None
    dy = torch.randn(n, d, device="cuda", generator=g).to(out)
    return x, w, b, dy


def _formula(x, w, b, dy, eps):
    x, w, dy = x.double(), w.double(), dy.double()
    mu = x.mean(-1, keepdim=True)
    rstd = ((x - mu).pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    xhat = (x - mu) * rstd
    y = xhat * w + (0 if b is None else b.double())
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return y, dx, (dy * xhat), dy, rstd, xhat, g


def _check(x, w, b, dy, got, eps=1e-5):
    y, dx, dw, db = got
    ry, rdx, dwt, dbt, rstd, xhat, g = _formula(x, w, b, dy, eps)
    n = x.shape[0]
    A = x.double().abs().amax(-1, keepdim=True) * rstd
    tol = 16 * U * ((A + xhat.abs()) * w.double().abs() + (0 if b is None else b.double().abs()))
    tol = tol + HALF_ULP[y.dtype] * ry.abs() * 1.01 + (2.0 ** -25 if y.dtype == torch.float16 else 0)
    assert ((y.double() - ry).abs() <= tol).all()
    tol = 64 * U * rstd * (1 + A) * g.abs().amax(-1, keepdim=True) * (1 + xhat.abs().amax(-1, keepdim=True))
    tol = tol + HALF_ULP[dx.dtype] * rdx.abs() * 1.01 + (2.0 ** -25 if dx.dtype == torch.float16 else 0)
    assert ((dx.double() - rdx).abs() <= tol).all()
    xerr = 16 * U * (A + xhat.abs()) * dy.double().abs()
    tol = 8 * U * n ** 0.5 * dwt.pow(2).sum(0).sqrt() + xerr.sum(0) + 1e-30
    assert ((dw.double() - dwt.sum(0)).abs() <= tol).all()
    if b is not None:
        tol = 8 * U * n ** 0.5 * dbt.pow(2).sum(0).sqrt() + 1e-30
        assert ((db.double() - dbt.sum(0)).abs() <= tol).all()


def _run(x, w, b, dy, out, eps=1e-5):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    b = b.detach().requires_grad_(True) if b is not None else None
    y = _layer_norm(x, w, b, eps=eps, out_dtype=out)
    assert y.dtype == out and y.is_contiguous()
    grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], dy)
    assert grads[0].dtype == x.dtype and grads[1].dtype == torch.float32
    return y.detach(), grads[0], grads[1], grads[2] if b is not None else None


# one row; widths below, at and above every split of a row over threads; odd widths; more rows than blocks
@pytest.mark.parametrize("n,d", [(1, 1), (3, 2), (1, 64), (7, 37), (5, 127), (33, 128), (64, 500), (300, 512), (17, 513),
                                 (9, 1024), (1300, 1037), (31, 2048), (12, 4100), (3, 8192), (5, 8196), (4, 9001),
                                 (3, 16384), (2, 16383), (5000, 256)])
def test_fp32_against_the_formula(n, d):
    x, w, b, dy = _inputs(n, d, torch.float32, torch.float32, seed=n + d)
    _check(x, w, b, dy, _run(x, w, b, dy, torch.float32))


@pytest.mark.parametrize("x_type,y_type", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                           (torch.float16, torch.float16), (torch.float32, torch.float16),
                                           (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("n,d", [(65, 768), (200, 2048), (19, 6144), (41, 1001), (3, 16384)])
def test_types(x_type, y_type, n, d):
    x, w, b, dy = _inputs(n, d, x_type, y_type, seed=d)
    _check(x, w, b, dy, _run(x, w, b, dy, y_type))


def test_without_bias():
    x, w, _, dy = _inputs(50, 640, torch.float32, torch.float32, bias=False)
    _check(x, w, None, dy, _run(x, w, None, dy, torch.float32))


@pytest.mark.parametrize("d", [2048, 333])
def test_rows_whose_mean_is_large_against_their_spread(d):
    x, w, b, dy = _inputs(20, d, torch.float32, torch.float32, shift=3000.0)
    _check(x, w, b, dy, _run(x, w, b, dy, torch.float32))


def test_constant_rows_give_the_bias():
    x = torch.full((4, 96), 2.5, device="cuda")
    w, b = torch.randn(96, device="cuda"), torch.randn(96, device="cuda")
    assert torch.equal(_layer_norm(x, w, b), b.expand(4, 96))


@pytest.mark.parametrize("d", [512, 511])
def test_strides_offsets_and_leading_shapes(d):
    x, w, b, dy = _inputs(24, 2 * d + 8, torch.bfloat16, torch.bfloat16)
    dy = dy[:, :d].contiguous()
    w, b = w[:d], b[:d]
    for view in (x[:, :d], x[:, 3:3 + d], x[::2, :d], x.t()[:d].t(), x[:, : 2 * d: 2]):
        g = dy[: view.shape[0]]
        _check(view, w, b, g, _run(view, w, b, g, torch.bfloat16))
    y3 = _layer_norm(x[:, :d].reshape(2, 3, 4, d), w, b)
    assert y3.shape == (2, 3, 4, d) and torch.equal(y3.view(24, d), _layer_norm(x[:, :d], w, b))
    y1 = _layer_norm(x[0, :d], w, b)
    assert y1.shape == (d,) and torch.equal(y1, y3.view(24, d)[0])
    # a gradient that is not dense: broadcast over rows, then transposed
    xx = x[:, :d].detach().clone().requires_grad_(True)
    y = _layer_norm(xx, w, b)
    for grad in (dy[:1].expand(24, d), dy.t().contiguous().t()):
        (dx,) = torch.autograd.grad(y, xx, grad, retain_graph=True)
        (want,) = torch.autograd.grad(y, xx, grad.contiguous(), retain_graph=True)
        assert torch.equal(dx, want)


def test_no_rows():
    x = torch.empty(0, 256, device="cuda", requires_grad=True)
    w, b = torch.ones(256, device="cuda", requires_grad=True), torch.zeros(256, device="cuda", requires_grad=True)
    y = _layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == (0, 256) and not dw.any() and not db.any()


def test_non_finite_rows_stay_in_their_row():
    x, w, b, dy = _inputs(8, 300, torch.float32, torch.float32)
    x[2, 5] = float("nan")
    x[4, 7] = float("inf")
    y = _layer_norm(x, w, b)
    bad = torch.zeros(8, dtype=torch.bool, device="cuda")
    bad[[2, 4]] = True
    assert torch.equal(~torch.isfinite(y).all(-1), bad)


def test_gradients_against_differences():
    """Directional differences of the kernel's own forward.  With h = 2^-8 the truncation is of order h^2 (2e-5 of
    the value), the rounding of y of order u / h (2e-5 of |y|, averaging out over the elements): 2e-3 is safe."""
    x, w, b, dy = _inputs(6, 200, torch.float32, torch.float32, seed=5)
    _, dx, dw, db = _run(x, w, b, dy, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(9)
    f = lambda *a: (_layer_norm(*a).double() * dy.double()).sum()  # noqa: E731
    h = 2.0 ** -8
    for which, grad in enumerate((dx, dw, db)):
        v = torch.randn(grad.shape, device="cuda", generator=g)
        v = v + grad / grad.norm() * v.norm()  # a direction along which the derivative is not small
        hi, lo = [x, w, b], [x, w, b]
        hi[which], lo[which] = hi[which] + h * v, lo[which] - h * v
        slope = (f(*hi) - f(*lo)) / (2 * h)
        want = (grad.double() * v.double()).sum()
        assert abs(slope - want) <= 2e-3 * abs(want)


def test_same_inputs_same_bits_and_other_streams():
    x, w, b, dy = _inputs(3000, 1024, torch.float32, torch.bfloat16)
    one = _run(x, w, b, dy, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = _run(x, w, b, dy, torch.bfloat16)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(one, two):
        assert torch.equal(p, q)


def test_refusals():
    x = torch.randn(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    with pytest.raises(ValueError, match="CUDA"):
        _layer_norm(x.cpu(), w.cpu())
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        _layer_norm(x.double(), w)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        _layer_norm(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="last dimension"):
        _layer_norm(torch.empty(2, 0, device="cuda"), torch.empty(0, device="cuda"))
    with pytest.raises(ValueError, match="last dimension"):
        _layer_norm(torch.empty(1, 16385, device="cuda"), torch.empty(16385, device="cuda"))
    with pytest.raises(ValueError, match="last dimension"):
        _layer_norm(torch.tensor(1.0, device="cuda"), w)
    with pytest.raises(ValueError, match="eps"):
        _layer_norm(x, w, eps=-1.0)
    with pytest.raises(RuntimeError, match="weight"):
        _layer_norm(x, w[:4])
    with pytest.raises(RuntimeError, match="weight"):
        _layer_norm(x, w.bfloat16())
    with pytest.raises(RuntimeError, match="bias"):
        _layer_norm(x, w, w.cpu())
    assert torch.isfinite(_layer_norm(x, w)).all()  # refused calls leave the context usable


# The backward kernels form first derivatives.  A second one, or a tangent, is refused and never left out of a sum.
@pytest.mark.parametrize("learned", ["x", "w", "b", "xwb"])
def test_second_derivatives_are_refused(learned):
    x, w, b, dy = _inputs(5, 96, torch.float32, torch.float32)
    leaves = [t.requires_grad_(True) for name, t in zip("xwb", (x, w, b)) if name in learned]
    want = torch.autograd.grad((_layer_norm(x, w, b) * dy).sum(), leaves)
    y = _layer_norm(x, w, b)
    grads = torch.autograd.grad((y * dy).sum(), leaves, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(grads, want))  # the first derivative itself is as ever
    penalty = sum(g.square().sum() for g in grads)
    for objective in (penalty, y.sum() + penalty):  # with and without another way to the inputs
        with pytest.raises(RuntimeError, match="layer_norm.*second derivative"):
            torch.autograd.grad(objective, leaves, retain_graph=True, allow_unused=True)
    objective = y.square().sum()
    objective.backward(create_graph=True)
    assert all(torch.isfinite(t.grad).all() for t in leaves)
    for t in leaves:
        t.grad = None


def test_a_factor_that_is_learned_gets_no_silent_gradient():
    x, w, b, dy = _inputs(5, 96, torch.float32, torch.float32)
    x.requires_grad_(True)
    s = torch.ones((), device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad((_layer_norm(x, w, b) * dy * s).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="layer_norm.*second derivative"):
        torch.autograd.grad(g.sum(), s, allow_unused=True)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("record", [False, True])
def test_tangents_are_refused(which, record):
    import torch.autograd.forward_ad as fwd
    args = list(_inputs(4, 64, torch.float32, torch.float32)[:3])
    if record:
        args = [t.requires_grad_(True) for t in args]
    with fwd.dual_level():
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="layer_norm.*forward-mode"):
            _layer_norm(*args)
