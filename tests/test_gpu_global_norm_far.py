"""Clipping by factors below the smallest normal fp32 value, 2^-126.

u = 2^-24: the factor carries the norm's rounding (2 u), its own division (2 u) and two products (u each), then half a step
of the type, or of its smallest value."""
import pytest
import torch

from gncde import engine

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.mark.parametrize("size,max_norm", [(1e37, 1e-6), (3e36, 1e-3), (1e37, 2.0 ** -126), (1e30, 1e-20), (1e37, 1e-44),
                                           (1e-3, 1e-42), (2.0 ** 127, 1e-30), (1.0, 2.0 ** -140), (1e-30, 1e-40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_factor_below_the_normal_values(dtype, size, max_norm):
    g = torch.Generator(device="cuda").manual_seed(0)
    ts = [((torch.rand(n, generator=g, device="cuda") - 0.5) * 2 * size / n ** 0.5).to(dtype) for n in (300, 1, 70001)]
    n = float(torch.cat([t.double() for t in ts]).square().sum().sqrt())
    max_norm = float(torch.tensor(max_norm))  # as fp32 holds it
    assert max_norm < n < 3.4e38
    out, stats = engine.clip_by_global_norm(ts, max_norm)
    assert abs(float(stats[0]) - n) <= 2 * U * n
    for t, o in zip(ts, out):
        w = t.double() * (max_norm / n)
        bound = (8 * U + HALF[dtype] * (1 + 8 * U)) * w.abs() + TINY[dtype]
        off = (o.double() - w).abs()
        assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} of the bound"
    place = [t.clone() for t in ts]
    engine.clip_by_global_norm(place, max_norm, out=place)
    assert all(torch.equal(a, b) for a, b in zip(place, out))


def test_half_values_by_a_tiny_factor():
    """fp16 values are too small to need such a factor for a result that is not zero."""
    t = [torch.full((64,), 60000.0, device="cuda", dtype=torch.float16), torch.full((4,), 3e37, device="cuda")]
    out, _ = engine.clip_by_global_norm(t, 1e-6)
    assert bool((out[0] == 0).all())
    n = float(torch.cat([x.double() for x in t]).square().sum().sqrt())
    assert bool(((out[1].double() - 3e37 * (1e-6 / n)).abs() <= 12 * U * 1e-6).all())
