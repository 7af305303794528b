"""Classes put out of reach by the type's lowest value in the bias (the finite form of -inf), in runs that fill whole tiles,
and logits as large everywhere.

u = 2^-24.  Where other classes are left, the lowest ones' terms are exact zeros and the bounds are those of the classes
left: logits |dl| <= (6 H + 16) u A, the softmax relative to its largest logit with 2 u (max l - min l) + 2^-23 + 256 u, and
sums over K terms (K + 64) u, as for any row."""
import pytest
import torch

from gncde import engine

pytestmark = pytest.mark.gpu
U, UB = 2.0 ** -24, 2.0 ** -8


def make(rows, hidden, classes, dtype, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = {"x": torch.randn(rows, hidden, generator=g, device="cuda"),
         "W": torch.randn(classes, hidden, generator=g, device="cuda") * hidden ** -0.5,
         "b": torch.randn(classes, generator=g, device="cuda")}
    c = {k: v.to(dtype) for k, v in c.items()}
    if kind == "rows":
        y = torch.rand(rows, classes, generator=g, device="cuda") ** 4
        c["t"] = y / y.sum(1, keepdim=True)
    else:
        c["t"] = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    c["g"] = torch.rand(rows, generator=g, device="cuda") * 2 - 0.5
    return c


SIZES = [(40, 8, 250), (40, 8, 500), (5, 300, 700), (40, 136, 1300), (300, 64, 2000), (600, 64, 30000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["i64", "rows"])
@pytest.mark.parametrize("size", SIZES)
def test_lowest_value_in_the_bias(size, kind, dtype):
    c = make(*size, dtype, kind)
    V, H = size[2], size[1]
    low = slice(V // 4, V)  # three quarters of the classes, whole tiles among them
    c["b"][low] = torch.finfo(dtype).min
    if kind == "rows":
        c["t"][:, low] = 0
    else:
        c["t"] %= V // 4
    x, W, b = (c[k].double() for k in ("x", "W", "b"))
    y = c["t"].double() if kind == "rows" else torch.zeros(size[0], V, dtype=torch.float64, device="cuda").scatter_(
        1, c["t"][:, None], 1.0)
    l, few = x @ W.T + b, slice(0, V // 4)
    A = (x.abs() @ W.abs().T + b.abs())[:, few].amax(1)
    S, lse = y.sum(1), torch.logsumexp(l, 1)
    yl = (y * l)[:, few]
    want = S * lse - yl.sum(1)
    d_l = (6 * H + 16) * U * A
    E = 4 * U * A + 2.0 ** -23 + 256 * U
    tol = S * (d_l + E) + d_l * S + (V / 64 + 64) * U * ((S * lse).abs() + yl.abs().sum(1))
    loss, stats = engine.linear_cross_entropy(c["x"], c["W"], c["b"], c["t"])
    assert bool(((loss.double() - want).abs() <= tol).all())
    gx, gW, gb = engine.linear_cross_entropy_grad(c["x"], c["W"], c["b"], c["t"], stats, c["g"])
    g = c["g"].double()
    p = torch.exp(l - lse[:, None])
    d = (g * S)[:, None] * p - g[:, None] * y
    ub = UB if dtype == torch.bfloat16 else U
    t_d = ((g * S).abs()[:, None] * p) * (2 * d_l + 2 * E)[:, None] + 4 * U * ((g * S).abs()[:, None] * p + g.abs()[:, None] * y)
    t_op = t_d + max(ub, 4 * U) * d.abs()
    for got, v, t, k in ((gx, d @ W, t_op @ W.abs() + (V + 64) * U * (d.abs() @ W.abs()), "gx"),
                         (gW, d.T @ x, t_op.T @ x.abs() + (size[0] + 64) * U * (d.abs().T @ x.abs()), "gW"),
                         (gb, d.sum(0), t_d.sum(0) + (size[0] + 64) * U * d.abs().sum(0), "gb")):
        # + the smallest step of a part of fp32 inputs, 2^-134, times the other factor
        bound = 1.01 * t + ub * (v.abs() + t) + 2.0 ** -120
        assert bool(((got.double() - v).abs() <= bound).all()), k
    assert bool((gW[low] == 0).all()) and bool((gb[low] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("base", ["lowest", -2.0 ** 100, -2.0 ** 40, -2.0 ** 31, 2.0 ** 31, 1.5 * 2.0 ** 31, 2.0 ** 100, "most"])
@pytest.mark.parametrize("size", [(40, 8, 256), (5, 300, 512), (40, 136, 1024), (300, 64, 32768)])
def test_rows_of_far_logits_are_finite(size, base, dtype):
    """Every logit of the row is the same far number: its loss (log V) is within fp32's rounding of that number, which may
    be all that is left of it, and nothing overflows on the way.  No gradient overflows."""
    c = make(*size, dtype, "i64")
    fi = torch.finfo(dtype)
    c["b"][:] = fi.min if base == "lowest" else fi.max if base == "most" else base
    far = float(c["b"][0].double().abs())
    loss, stats = engine.linear_cross_entropy(c["x"], c["W"], c["b"], c["t"])
    assert bool((loss.abs() <= 16 + 8 * U * far).all())
    for t in engine.linear_cross_entropy_grad(c["x"], c["W"], c["b"], c["t"], stats, c["g"]):
        assert bool(torch.isfinite(t).all())
