"""The read-out's cross-entropy where every logit is a whole number that all its sums hold exactly: what is left is the
softmax, far from zero.

Inputs: x and W whole numbers up to 3, W for a few of the hidden values only, the bias a constant B and whole numbers up to
8: |l - B| <= D, every partial sum a whole number below 2^24, exact in any order and in either type.  With the logits exact,
u = 2^-24:
  exponent's argument  (l - top) log2 e within 2 u of itself, l - top and top - lse' being exact or rounded once
  sum of exponentials  relative error <= (4 D + 4 + 256) u: the arguments', the exponential's own (2 u each time it is
                       taken, twice here) and those of 256 additions; an error as large in its logarithm
  loss                 S times that, + (V / 64 + 64) u sum |y| (top - l), + half a step of the largest term: nothing that
                       grows with B
  dl                   |g| S p times the above, once for the sum and once for the exponential, + 4 u (|g| S p + |g y|)
  gb                   fp32: the sums' (R + 64) u sum |dl| more, and half a step of its type
A loss that subtracts two numbers of B's size is off by u B = 2^-8 at B = 65536, a thousand times the bound."""
import pytest
import torch

from gncde import engine

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def make(rows, hidden, classes, dtype, kind, base, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=g, device="cuda").float()

    W = whole(-3, 3, classes, hidden)
    W[:, 4:] = 0
    c = {"x": whole(-3, 3, rows, hidden), "W": W, "b": base * torch.ones(classes, device="cuda")}
    # bf16 holds 65536 and 1024 and few numbers beside them: the small part of the bias goes into a hidden value of one
    c["x"][:, 0] = 1
    c["W"][:, 0] = whole(-8, 8, classes)
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    c["x"][::2, 1:4] = c["W"][t[::2], 1:4].sign() * 3  # every other row is fairly sure of its class
    if kind == "rows":
        y = torch.rand(rows, classes, generator=g, device="cuda") ** 8
        y *= torch.rand(rows, 1, generator=g, device="cuda") * 2 / y.sum(1, keepdim=True)
        y[::2] = 0
        y[torch.arange(0, rows, 2, device="cuda"), t[::2]] = 1.0
        t = y
    c = {k: v.to(dtype) for k, v in c.items()}
    c["t"], c["g"] = t, torch.rand(rows, generator=g, device="cuda") * 2 - 0.5
    return c


CASES = [(40, 8, 30), (300, 32, 255),                       # few classes
         (1, 40, 700), (5, 300, 700), (16, 64, 5000),      # few rows
         (40, 136, 513), (300, 64, 2000), (700, 200, 9001)]  # tiles


@pytest.mark.parametrize("base", [0.0, 1024.0, -65536.0, 65536.0, -2.0 ** 22])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["i64", "rows"])
@pytest.mark.parametrize("size", CASES)
def test_loss_far_from_zero(size, kind, dtype, base):
    c = make(*size, dtype, kind, base)
    R, H, V = size
    l = c["x"].double() @ c["W"].double().T + c["b"].double()
    assert bool((l == l.round()).all()) and float(l.abs().max()) < 2 ** 23
    y = c["t"].double() if kind == "rows" else torch.zeros_like(l).scatter_(1, c["t"][:, None], 1.0)
    S, top = y.sum(1), l.amax(1, keepdim=True)
    D = float((top - l).max())
    d_log = (4 * D + 260) * U
    want = S * torch.logsumexp(l - top, 1) + (y * (top - l)).sum(1)
    tol = S * d_log + (V / 64 + 64) * U * (y * (top - l)).sum(1) + U * (S * torch.logsumexp(l - top, 1) + want)
    loss, _ = engine.linear_cross_entropy(c["x"], c["W"], c["b"], c["t"])
    off = (loss.double() - want).abs()
    assert bool((off <= tol).all()), f"{float((off / tol).max()):.3g} of the bound"
    assert bool((loss >= 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("base", ["lowest", -2.0 ** 100, -2.0 ** 40, -2.0 ** 32, 2.0 ** 32, 1.5 * 2.0 ** 33, 2.0 ** 100, "most"])
@pytest.mark.parametrize("kind", ["i64", "rows"])
@pytest.mark.parametrize("size", [(40, 8, 256), (5, 300, 512), (40, 136, 1024), (300, 64, 32768)])
def test_loss_of_equal_logits(size, kind, base, dtype):
    """The products, below 2^7, vanish in fp32's rounding of the bias (half a step of 2^8 and more): all V logits are the
    same number, the sum of exponentials is V exactly and the loss S log V, within the logarithm's 2 u, one product's
    rounding, and that of S: V / 64 + 64 additions in the kernel, 64 bits here."""
    c = make(*size, dtype, kind, 0.0)
    fi = torch.finfo(dtype)
    c["b"][:] = fi.min if base == "lowest" else fi.max if base == "most" else base
    assert float((c["x"].float().abs() @ c["W"].float().abs().T).max()) < 2 ** 7
    S = c["t"].double().sum(1) if kind == "rows" else torch.ones(size[0], dtype=torch.float64, device="cuda")
    want = S * torch.log(torch.tensor(float(size[2]), dtype=torch.float64))
    loss, _ = engine.linear_cross_entropy(c["x"], c["W"], c["b"], c["t"])
    assert bool(((loss.double() - want).abs() <= (size[2] / 64 + 68) * U * want).all())


def _grads(c, need=(True, True, True)):
    _, stats = engine.linear_cross_entropy(c["x"], c["W"], c["b"], c["t"])
    return engine.linear_cross_entropy_grad(c["x"], c["W"], c["b"], c["t"], stats, c["g"], None, *need)


def _check_grads(c, l, y, p, D):
    """gx, gW and gb against the formula: of dl, |g| S p carries (8 D + 360) u: the sum's (4 D + 260) u, the exponent's 4 u of
    l - lse, which is below D + log V, 6 u of three exponentials and 4 u of the products; then the operand's rounding (bf16:
    half a step of dl) and the sums'."""
    R, V = l.shape
    bf = c["x"].dtype == torch.bfloat16
    half = 2.0 ** -8 if bf else U
    g, S, x, W = c["g"].double()[:, None], y.sum(1, keepdim=True), c["x"].double(), c["W"].double()
    gp, d = (g * S).abs() * p, g * (S * p - y)
    t_d = gp * (8 * D + 360) * U + 4 * U * (gp + g.abs() * y)
    t_op = t_d + max(half, 4 * U) * (d.abs() + t_d) + 2.0 ** -134
    for name, got, v, t in zip(("gx", "gW", "gb"), _grads(c), (d @ W, d.T @ x, d.sum(0)),
                               (t_op @ W.abs() + (V + 64) * U * (d.abs() @ W.abs()),
                                t_op.T @ x.abs() + (R + 64) * U * (d.abs().T @ x.abs()),
                                t_d.sum(0) + (R + 64) * U * d.abs().sum(0))):
        off, tol = (got.double() - v).abs(), 1.01 * t + half * (v.abs() + t) + 2.0 ** -126
        assert bool((off <= tol).all()), f"{name}: {float((off / tol).max()):.3g} of the bound"


@pytest.mark.parametrize("base", [0.0, 1024.0, -65536.0, 65536.0, -2.0 ** 22])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["i64", "rows"])
@pytest.mark.parametrize("size", CASES)
def test_gradients_far_from_zero(size, kind, dtype, base):
    c = make(*size, dtype, kind, base)
    l = c["x"].double() @ c["W"].double().T + c["b"].double()
    y = c["t"].double() if kind == "rows" else torch.zeros_like(l).scatter_(1, c["t"][:, None], 1.0)
    top = l.amax(1, keepdim=True)
    _check_grads(c, l, y, torch.softmax(l - top, 1), float((top - l).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("base", ["lowest", -2.0 ** 100, -2.0 ** 32, 2.0 ** 32, 1.5 * 2.0 ** 33, 2.0 ** 100, "most"])
@pytest.mark.parametrize("kind", ["i64", "rows"])
@pytest.mark.parametrize("size", [(40, 8, 256), (5, 300, 512), (40, 136, 1024), (300, 64, 32768)])
def test_gradients_of_equal_logits(size, kind, base, dtype):
    """All V logits the same far number: p = 1 / V, which lse, rounded to a step of that number, does not hold by itself."""
    c = make(*size, dtype, kind, 0.0)
    fi = torch.finfo(dtype)
    c["b"][:] = fi.min if base == "lowest" else fi.max if base == "most" else base
    R, H, V = size
    l = torch.zeros(R, V, dtype=torch.float64, device="cuda")
    y = c["t"].double() if kind == "rows" else torch.zeros_like(l).scatter_(1, c["t"][:, None], 1.0)
    _check_grads(c, l, y, torch.full_like(l, 1 / V), 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["i64", "rows"])
@pytest.mark.parametrize("size", [(40, 8, 30), (5, 300, 700), (40, 136, 513)])
def test_rows_that_nothing_can_be(size, kind, dtype):
    """-inf in the whole bias: the softmax of no class is not a number, and neither is what it enters."""
    c = make(*size, dtype, kind, 0.0)
    c["b"][:] = -float("inf")
    assert bool(torch.isnan(engine.linear_cross_entropy(c["x"], c["W"], c["b"], c["t"])[0]).all())
    gx, gW, gb = _grads(c)
    assert bool(torch.isnan(gx).all()) and bool(torch.isnan(gb).all()) and bool(torch.isnan(gW).all())
