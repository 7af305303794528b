"""The read-out's cross-entropy (gncde_linear_cross_entropy, .._grad) against the formula in 64 bits.

Tolerances are bounds, worked out from the arithmetic and computed in 64 bits beside each reference:
  u = 2^-24 (fp32), ub = 2^-8 (bf16: half a step relative to the value).
  logits   |dl| <= (6 H + 16) u A, A_rv = sum_h |x_rh W_vh| + |b_v|: products are exact (bf16) or leave 4 u of |x||W|
           (three parts), at most 6 H fp32 additions, the bias added once.
  lse      |dlse| <= max_v |dl| + E with E = 2 u (max_v l - min_v l over the classes that matter: bounded by 2 max A)
           for the exponent's argument + 2^-23 for the exponential + 256 u for the sums (32 terms a lane, then 2 + 3
           levels, then one level a tile of 128 classes and 64 lanes: below 256 additions in any order here).
  loss     |S| dlse + sum |y| |dl| + (V/64 + 64) u (|S lse| + sum |y l|)
  dl       |d(dl)| <= |g| S p (|dl| + |dlse| + E) + u (|g| S p + |g y|) (+ ub |dl| rounded to bf16 operands, or 4 u)
  parts    fp32 inputs: the last part ends at bf16's smallest step 2^-133, so each of x, W and dl is off by at most 2^-134
           whatever its size: the product's other factor times that (it shows only where a factor is near 2^127).
  sums     + (K + 64) u sum |dl| |factor| over the K terms, + half a step of the result's type.  Where that sum of
           magnitudes reaches fp32's largest value, a partial sum may pass it: not a finite value then.
"""
import math

import pytest
import torch

from gncde import autograd, engine

pytestmark = pytest.mark.gpu
U, UB = 2.0 ** -24, 2.0 ** -8


def make(rows, hidden, classes, dtype, kind="i64", bias=True, masked=True, seed=0, scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = {}
    c["x"] = torch.randn(rows, hidden, generator=g, device="cuda").to(dtype)
    c["W"] = (torch.randn(classes, hidden, generator=g, device="cuda") * (scale / math.sqrt(hidden))).to(dtype)
    c["b"] = (0.5 * torch.randn(classes, generator=g, device="cuda")).to(dtype) if bias else None
    if kind == "rows":
        y = torch.rand(rows, classes, generator=g, device="cuda") ** 4
        y *= torch.rand(rows, 1, generator=g, device="cuda") * 2 / y.sum(1, keepdim=True)
        if rows > 2:
            y[1] = 0.0  # a row without any mass
        c["target"] = y
    else:
        t = torch.randint(0, classes, (rows,), generator=g, device="cuda")
        if rows > 3:
            t[0], t[-1] = classes - 1, 0
            t[2] = -100
        c["target"] = t.to(torch.int32 if kind == "i32" else torch.int64)
    c["mask"] = torch.rand(rows, generator=g, device="cuda") < 0.7 if masked else None
    c["g"] = torch.rand(rows, generator=g, device="cuda") * 2 - 0.5
    return c


def reference(c):
    """Loss and gradients in 64 bits, with the bounds of the module's docstring."""
    x, W = c["x"].double(), c["W"].double()
    R, H = x.shape
    V = W.shape[0]
    bf = c["x"].dtype == torch.bfloat16
    b = c["b"].double() if c["b"] is not None else torch.zeros(V, dtype=torch.float64, device=x.device)
    keep = torch.ones(R, dtype=torch.bool, device=x.device) if c["mask"] is None else c["mask"].clone()
    soft = c["target"].dtype == torch.float32
    if soft:
        y = c["target"].double()
    else:
        t = c["target"].long()
        keep &= t >= 0
        y = torch.zeros(R, V, dtype=torch.float64, device=x.device)
        y.scatter_(1, t.clamp(0, V - 1).unsqueeze(1), 1.0)
    x = torch.where(keep[:, None], x, torch.zeros_like(x))
    y = torch.where(keep[:, None], y, torch.zeros_like(y))
    g = torch.where(keep, c["g"].double(), torch.zeros(R, dtype=torch.float64, device=x.device))
    l = x @ W.T + b
    A = x.abs() @ W.abs().T + torch.where(torch.isinf(b), torch.zeros_like(b), b.abs())
    lse = torch.logsumexp(l, 1)
    S = y.sum(1)
    yl = torch.where(y == 0, torch.zeros_like(l), y * l)
    loss = torch.where(keep, S * lse - yl.sum(1), torch.zeros_like(lse))
    end = 0.0 if bf else 2.0 ** -134
    dl_l = (6 * H + 16) * U * A + end * (x.abs().sum(1)[:, None] + W.abs().sum(1)[None, :])
    E = 2 * U * 2 * A.amax(1) + 2.0 ** -23 + 256 * U
    d_lse = dl_l.amax(1) + E
    tol_loss = S.abs() * d_lse + (y.abs() * dl_l).sum(1) + (V / 64 + 64) * U * ((S * lse).abs() + yl.abs().sum(1))
    p = torch.exp(l - lse[:, None])
    gp = (g * S).abs()[:, None] * p
    d = (g * S)[:, None] * p - g[:, None] * y
    tol_d = gp * (dl_l + (d_lse + E)[:, None]) + 4 * U * (gp + (g[:, None] * y).abs())
    tol_op = tol_d + (UB if bf else 4 * U) * d.abs() + end
    out = {"loss": (loss, tol_loss + 1e-30), "lse": torch.where(keep, lse, torch.zeros_like(lse))}
    half = UB if bf else U
    for name, v, tol, k in (
            ("gx", d @ W, tol_op @ W.abs() + (V + 64) * U * (d.abs() @ W.abs()) + end * d.abs().sum(1)[:, None], V),
            ("gW", d.T @ x, tol_op.T @ x.abs() + (R + 64) * U * (d.abs().T @ x.abs()) + end * d.abs().sum(0)[:, None], R),
            ("gb", d.sum(0), tol_d.sum(0) + (R + 64) * U * d.abs().sum(0), R)):
        out[name] = (v, tol * 1.01 + half * (v.abs() + tol) + 1e-30)
    out["gx"] += (d.abs() @ W.abs(),)
    out["gW"] += (d.abs().T @ x.abs(),)
    return out


def close(got, want, name):
    v, tol, *most = want  # most: the largest magnitude a partial sum can have
    off = (got.double() - v).abs()
    bad = ~(off <= tol)
    if most:
        bad &= ~((most[0] >= torch.finfo(torch.float32).max) & ~torch.isfinite(got))
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / tol).max()):.3g} of its bound"


def call(c, need=(True, True, True)):
    loss, stats = engine.linear_cross_entropy(c["x"], c["W"], c["b"], c["target"], c["mask"])
    gs = engine.linear_cross_entropy_grad(c["x"], c["W"], c["b"], c["target"], stats, c["g"], c["mask"], *need)
    return loss, stats, gs


def check(c):
    ref = reference(c)
    loss, stats, (gx, gW, gb) = call(c)
    close(loss, ref["loss"], "loss")
    assert gx.dtype == gW.dtype == c["x"].dtype
    close(gx, ref["gx"], "gx")
    close(gW, ref["gW"], "gW")
    if c["b"] is not None:
        close(gb, ref["gb"], "gb")
    else:
        assert gb is None


SIZES = [(1, 1, 1), (1, 16, 2), (3, 5, 7), (2, 64, 64), (17, 32, 255), (130, 64, 129), (255, 32, 255), (64, 200, 5000),
         (257, 96, 513), (300, 333, 1001), (1030, 72, 4099),
         # everything in LDS, at its widths and past one workgroup a CU
         (40, 48, 100), (33, 128, 60), (100, 16, 440), (5000, 20, 70), (21, 80, 130), (50, 3, 500),
         # few rows
         (1, 512, 4096), (16, 100, 700), (13, 333, 1234), (5, 1000, 77), (2, 40, 9001), (4, 2050, 300),
         (16, 4000, 90)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind", ["i64", "rows"])
def test_against_64_bits(size, dtype, kind):
    check(make(*size, dtype, kind))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_index32_without_bias_and_mask(dtype):
    check(make(65, 40, 300, dtype, "i32", bias=False, masked=False))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,kind", [((300, 64, 52000), "i64"), ((10300, 1100, 130), "rows")])
def test_large_tiles(size, kind, dtype):
    check(make(*size, dtype, kind))


@pytest.mark.parametrize("rows,dtype,kind", [(12000, torch.float32, "i64"), (12000, torch.float32, "rows"),
                                             (33000, torch.bfloat16, "i64"), (33000, torch.bfloat16, "rows")])
def test_classes_in_several_pieces(rows, dtype, kind):
    """So many rows that dl of all classes passes 1 GiB: the gradient takes the classes in pieces, the last one ragged."""
    check(make(rows, 40, 17001, dtype, kind))


@pytest.mark.parametrize("rows", [1, 2, 16, 17, 40])
def test_few_rows(rows):
    check(make(rows, 512, 40000, torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("classes", [1, 2, 3, 4, 5, 130, 257, 510, 515])
def test_label_rows_at_the_last_classes(classes, dtype):
    """A wide hidden row (tiled kernels) and label rows whose last classes end anywhere within four."""
    check(make(40, 300, classes, dtype, "rows"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,classes", [(31, 513), (32, 545), (33, 543), (63, 608), (64, 577), (65, 639), (97, 640),
                                          (129, 1025), (255, 1055), (256, 1056), (257, 1057)])
def test_rows_and_classes_around_the_steps(rows, classes, dtype):
    """Contractions that end anywhere within the steps of gx (classes) and gW (rows)."""
    check(make(rows, 136, classes, dtype))


def test_label_rows_without_mask_are_read_as_they_lie():
    """Rows that start on 16 bytes and of which none can be left out."""
    check(make(70, 64, 700, torch.bfloat16, "rows", masked=False))


@pytest.mark.parametrize("hidden", [64, 72, 333])
def test_hidden_gradient_alone_with_rows_left_out(hidden):
    """NaN in the rows left out, and no gradient of the weights that would put them aside."""
    c = make(100, hidden, 700, torch.bfloat16)
    c["mask"][5:40] = False
    want = call(c)[2][0]
    x = c["x"].clone()
    x[5:40] = float("nan")
    got = call(dict(c, x=x), (True, False, False))[2][0]
    assert torch.equal(got, want) and bool((got[5:40] == 0).all())


def test_large_logits():
    """Logits in the hundreds: the largest carries all the mass and nothing overflows."""
    for dtype in (torch.float32, torch.bfloat16):
        check(make(70, 64, 500, dtype, scale=200.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["i64", "rows"])
def test_rows_left_out_change_nothing(dtype, kind):
    """NaN and inf in the hidden rows, labels and cotangents of rows left out."""
    c = make(200, 48, 300, dtype, kind)
    c["mask"][:3] = False
    ref = call(c)
    d = dict(c)
    out = ~c["mask"]
    if kind == "i64":
        out |= c["target"] < 0
    fill = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")
    for k in ("x", "g"):
        d[k] = c[k].clone()
        n = int(out.sum())
        v = fill[torch.arange(n, device="cuda") % 3]
        d[k][out] = v.to(d[k].dtype)[:, None].expand(n, 48) if k == "x" else v
    if kind == "rows":
        d["target"] = c["target"].clone()
        d["target"][out] = float("nan")
    got = call(d)
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
    assert bool((got[0][out] == 0).all()) and bool((got[2][0][out] == 0).all())
    for a, b in zip(ref[2], got[2]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_row_left_out(dtype):
    c = make(50, 24, 90, dtype)
    c["mask"][:] = False
    loss, stats, (gx, gW, gb) = call(c)
    for t in (loss, stats, gx, gW, gb):
        assert bool((t == 0).all())


def test_classes_that_nothing_can_be():
    """-inf in the bias: no mass there, no gradient, whole tiles of classes among them."""
    c = make(90, 32, 700, torch.float32)
    c["b"][100:420] = -float("inf")
    c["target"][:] = torch.where((c["target"] >= 100) & (c["target"] < 420), torch.full_like(c["target"], 5), c["target"])
    check_finite = reference(c)
    loss, _, (gx, gW, gb) = call(c)
    close(loss, check_finite["loss"], "loss")
    close(gx, check_finite["gx"], "gx")
    close(gW, check_finite["gW"], "gW")
    assert bool((gW[100:420] == 0).all()) and bool((gb[100:420] == 0).all())
    y = make(90, 32, 700, torch.float32, "rows")
    y["b"] = c["b"]
    y["target"][:, 100:420] = 0
    close(call(y)[0], reference(y)["loss"], "loss")


def test_values_near_the_largest():
    """fp32 values whose leading bf16 part would round to infinity stay finite."""
    c = make(40, 8, 30, torch.float32)
    c["x"].zero_()
    c["x"][:, 0] = 3.4e38
    c["W"].mul_(1e-38)
    check(c)


def test_index_past_the_last_class_is_nan():
    c = make(40, 16, 30, torch.float32, masked=False)
    c["target"][5] = 30
    loss, stats, (gx, gW, gb) = call(c)
    assert bool(torch.isnan(loss[5])) and int(torch.isnan(loss).sum()) == 1
    assert bool(torch.isnan(gx[5]).all()) and bool(torch.isnan(gW).all()) and bool(torch.isnan(gb).all())
    assert int(torch.isnan(gx).any(1).sum()) == 1


def test_no_rows():
    c = make(1, 16, 30, torch.bfloat16)
    c = {**c, "x": c["x"][:0], "target": c["target"][:0], "mask": c["mask"][:0], "g": c["g"][:0]}
    loss, stats, (gx, gW, gb) = call(c)
    assert loss.shape == (0,) and stats.shape == (0, 2) and gx.shape == (0, 16)
    assert bool((gW == 0).all()) and bool((gb == 0).all())


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (False, False, False)])
def test_only_the_gradients_asked_for(need):
    c = make(100, 40, 300, torch.bfloat16)
    full = call(c)[2]
    for want, a, b in zip(need, call(c, need)[2], full):
        assert (a is None) if not want else torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """Leading axes, strided views and addresses off 16 bytes give what contiguous tensors give."""
    c = make(60, 40, 130, dtype)
    ref = call(c)
    lead = dict(c, x=c["x"].view(3, 4, 5, 40), target=c["target"].view(3, 4, 5), mask=c["mask"].view(3, 4, 5),
                g=c["g"].view(3, 4, 5))
    got = call(lead)
    assert got[0].shape == (3, 4, 5) and got[1].shape == (3, 4, 5, 2) and got[2][0].shape == (3, 4, 5, 40)
    assert torch.equal(got[0].flatten(), ref[0])
    for a, b in zip(got[2], ref[2]):
        assert torch.equal(a.flatten(), b.flatten())
    strided = dict(c, x=c["x"].t().contiguous().t(), W=c["W"].t().contiguous().t(),
                   g=torch.stack([c["g"], c["g"]], 1)[:, 0])
    off = {}
    for k in ("x", "W"):
        buf = torch.empty(c[k].numel() + 1, dtype=dtype, device="cuda")
        off[k] = buf[1:].view(c[k].shape)
        off[k].copy_(c[k])
    for d in (strided, dict(c, **off), dict(c, x=off["x"]), dict(c, W=off["W"])):
        got = call(d)
        assert torch.equal(got[0], ref[0])
        for a, b in zip(got[2], ref[2]):
            assert torch.equal(a, b)


class _NotPlain:
    """The compiled calls turning every call down: what is left is the Python code behind them."""
    readout_loss = readout_grad = tensor_list = staticmethod(lambda *a: None)


@pytest.mark.parametrize("kind", ["i32", "i64", "rows"])
def test_compiled_and_python_calls_agree(kind, monkeypatch):
    c = make(70, 48, 400, torch.bfloat16, kind)
    n = dict(c, b=None, mask=None)
    want = [call(c), call(n), call(c, (True, False, False))]
    monkeypatch.setattr(engine, "_fast", _NotPlain)
    got = [call(c), call(n), call(c, (True, False, False))]
    for w, o in zip(want, got):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])
        for a, b in zip(w[2], o[2]):
            assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


def test_repeatable():
    c = make(700, 64, 5000, torch.bfloat16, "rows")
    a, b = call(c), call(c)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


def test_streams_and_two_calls_at_once():
    cs = [make(500, 64, 3000, torch.float32, seed=1), make(400, 128, 2000, torch.bfloat16, "rows", seed=2)]
    want = [call(c) for c in cs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(call(c))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        w = want[i % 2]
        assert torch.equal(r[0], w[0]) and all(torch.equal(a, b) for a, b in zip(r[2], w[2]))


def test_captured_and_replayed():
    """Loss and gradient in one graph, replayed on new inputs with eager work between; two graphs hold their own
    workspaces."""
    cs = [make(300, 64, 2000, torch.bfloat16, seed=3), make(300, 64, 2000, torch.float32, "rows", seed=4)]
    for c in cs:
        call(c)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    for k in range(3):
        for c in cs:
            c["x"].copy_(torch.randn_like(c["x"]))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for c, o in zip(cs, outs):
            w = call(c)
            assert torch.equal(o[0], w[0]) and all(torch.equal(a, b) for a, b in zip(o[2], w[2]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd(dtype):
    c = make(120, 40, 300, dtype)
    x, W, b = (c[k].clone().requires_grad_() for k in ("x", "W", "b"))
    loss = autograd.linear_cross_entropy(x, W, b, c["target"], c["mask"])
    assert loss.shape == (120,) and loss.dtype == torch.float32
    got = torch.autograd.grad((loss * c["g"]).sum(), (x, W, b))
    for a, w in zip(got, call(c)[2]):
        assert torch.equal(a, w)
    loss = autograd.linear_cross_entropy(x, W.detach(), None, c["target"], None)
    (gx,) = torch.autograd.grad(loss.sum(), (x,))
    ones = torch.ones(120, device="cuda")
    _, stats = engine.linear_cross_entropy(c["x"], c["W"], None, c["target"])
    assert torch.equal(gx, engine.linear_cross_entropy_grad(c["x"], c["W"], None, c["target"], stats, ones)[0])


def test_gradient_against_differences():
    """Central differences of the operator's own loss along random directions.  The third derivative along a direction
    that moves row r's logits by at most m_r a unit is below S m^3 (a third central moment of values in an interval of
    length 2 m is below 2 m^3, S being the row's mass), so the difference is off by e^2 / 6 of 2 S m^3, and by the
    losses' own bounds over e."""
    for kind in ("i64", "rows"):
        c = make(24, 16, 40, torch.float32, kind)
        c["g"].fill_(1.0)
        keep = c["mask"] if kind == "rows" else c["mask"] & (c["target"] >= 0)
        S = c["target"].sum(1).double() if kind == "rows" else torch.ones(24, dtype=torch.float64, device="cuda")
        ref = reference(c)
        gx, gW, gb = call(c)[2]
        e = 2.0 ** -7
        for key, grad in (("x", gx), ("W", gW), ("b", gb)):
            g = torch.Generator(device="cuda").manual_seed(9)
            d = torch.randn(c[key].shape, generator=g, device="cuda")
            move = {"x": lambda: d.double() @ c["W"].double().T, "W": lambda: c["x"].double() @ d.double().T,
                    "b": lambda: d.double().expand(24, 40)}[key]().abs().amax(1)
            f = []
            for s in (e, -e):
                z = dict(c)
                z[key] = c[key] + s * d
                f.append(float(engine.linear_cross_entropy(z["x"], z["W"], z["b"], z["target"], z["mask"])[0].double().sum()))
            diff = (f[0] - f[1]) / (2 * e)
            exact = float((grad.double() * d.double()).sum())
            tol = float((e ** 2 / 6 * 2 * S * move ** 3 * keep).sum()) + 2 * float(ref["loss"][1].sum()) / e + \
                float((ref["g" + key][1] * d.double().abs()).sum())
            # the moved argument is rounded once: u |value| a logit's factor
            tol += float((U / e * S * keep * 4 * (c["x"].double().abs() @ c["W"].double().abs().T + 2).amax(1)).sum())
            assert abs(diff - exact) <= tol, (key, diff, exact, tol)
            # the bound says something: far below the change that a gradient of this size makes along d
            assert tol < 0.1 * float(grad.double().norm() * d.double().norm()), tol


def test_training_step_of_the_tgb_model():
    """The fused read-out loss in TGBGraphNeuralCDE, through make_step with ClippedOptimiser: the same loss and
    parameter gradients as the materialised logits give, and the same update as torch's clipping."""
    from gncde import train
    from gncde.models import TGBGraphNeuralCDE, vector_fields
    n, h, de, B, T = 12, 8, 4, 2, 4
    g = torch.Generator().manual_seed(5)
    ts = torch.linspace(0, 1, T).repeat(B, 1)
    A = torch.rand(B, T, n, n, generator=g) * 0.2
    X = torch.stack([ts[:, :, None, None].expand_as(A), A], dim=-1).to("cuda")
    co = engine.hermite_coefficients(ts.to("cuda"), X)
    coeffs = tuple(co[:, :, q].contiguous() for q in range(4))
    x_data, x0 = torch.rand(B, T, n, n, generator=g), torch.rand(B, n, n, generator=g)
    labels = torch.rand(B, n, n, generator=g)
    mask = torch.rand(B, n, generator=g) < 0.6

    def model(readout):
        vf = vector_fields.PermEquivGraphVectorField(input_dim=h, hidden_dim=h, output_dim=h * de * 2, num_layers=2,
                                                     data_embed_dim=de, num_nodes=n, key=3)
        return TGBGraphNeuralCDE({"hidden_dim": h}, vf, "cubic", 3, dt0=0.1, readout_loss=readout).to("cuda")

    res = {}
    for readout in ("logits", "fused"):
        m = model(readout)
        loss, count = m.loss_terms(ts, coeffs, x_data, x0, labels, mask)
        loss.backward()
        res[readout] = (float(loss.detach()), float(count), [None if p.grad is None else p.grad.clone() for p in m.parameters()])
    assert res["logits"][1] == res["fused"][1] == float(mask.sum())
    # both are fp32 evaluations of the same sums over n = 12 classes and 24 rows: 2^-24 times a few hundred additions
    assert abs(res["logits"][0] - res["fused"][0]) <= 2.0 ** -14 * abs(res["logits"][0])
    # The data encoder's bias moves every knot alike, so its gradient is a difference of equal sums: rounding alone, at
    # most 2^-24 of B T n de < 2^10 summands, each within the largest parameter gradient.
    largest = max(float(a.norm()) for a in res["logits"][2] if a is not None)
    for a, b in zip(res["logits"][2], res["fused"][2]):
        assert (a is None) == (b is None)
        if a is not None:
            assert float((a - b).norm()) <= 2.0 ** -12 * float(a.norm()) + 2.0 ** -14 * largest

    m, ref = model("fused"), model("fused")
    opt = train.ClippedOptimiser(torch.optim.AdamW(m.parameters(), lr=1e-2, weight_decay=1e-3), max_norm=0.05)
    got = train.make_step(opt, m.loss_terms, ts, coeffs, x_data, x0, labels, mask)
    loss, count = ref.loss_terms(ts, coeffs, x_data, x0, labels, mask)
    (loss / count).backward()
    for p in ref.parameters():
        if p.grad is None:
            p.grad = torch.zeros_like(p)
    norm = torch.sqrt(sum((p.grad.double() ** 2).sum() for p in ref.parameters()))
    assert float(norm) > 0.05
    top = max(float(p.grad.abs().max()) for p in ref.parameters())
    for p in ref.parameters():
        p.grad.mul_((0.05 / norm).float())
    before = [p.detach().clone() for p in ref.parameters()]
    torch.optim.AdamW(ref.parameters(), lr=1e-2, weight_decay=1e-3).step()
    assert abs(float(got[0]) - float((loss / count).detach())) <= 1e-6 * abs(float((loss / count).detach()))
    assert abs(float(got[1]) - top) <= 1e-5 * top
    most = max(float((p.detach() - q).abs().max()) for p, q in zip(ref.parameters(), before))
    assert abs(float(got[2]) - most) <= 1e-3 * most
    # Adam's first step is lr g / (|g| + 1e-8): for |g| > 1e-4 it is lr sign(g) to 1e-4 of lr.  A gradient below the
    # rounding bound above may have either sign: two steps of lr between them.
    scale = 0.05 / float(norm)
    for p, q in zip(m.parameters(), ref.parameters()):
        off = (p.detach() - q.detach()).abs()
        sure = q.grad.abs() > max(1e-4, 2.0 ** -13 * largest * scale)
        assert bool((off <= torch.where(sure, 1e-2 * 2e-4 + 2.0 ** -22, 2.02e-2)).all())
