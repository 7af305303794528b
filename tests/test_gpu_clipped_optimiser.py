"""train.ClippedOptimiser: what it does to its arguments, and gradients that lie in memory in other orders."""
import pytest
import torch

from gncde import engine, train

pytestmark = pytest.mark.gpu


def params(seed=3):
    """fp32 and bf16 parameters; the third is a transposed view's copy that keeps its strides."""
    g = torch.Generator().manual_seed(seed)
    out = [torch.nn.Parameter(torch.randn(s, generator=g).to("cuda", dt)) for s, dt in
           (((20, 30), torch.float32), ((8, 8), torch.bfloat16), ((1,), torch.float32))]
    out.insert(2, torch.nn.Parameter(torch.randn(7, 40, generator=g).to("cuda").t()))
    assert not out[2].is_contiguous()
    return out


def flat(ps, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(sum(p.numel() for p in ps), generator=g, device="cuda")


@pytest.mark.parametrize("max_norm", [0.5, 1e6, None])
def test_step_leaves_the_flat_gradient(max_norm):
    """The flat gradient is the caller's: fp32 parameters' pieces of it are not clipped in place."""
    ps = params()
    opt = train.ClippedOptimiser(torch.optim.SGD(ps, lr=0.1), max_norm)
    f = flat(ps)
    keep = f.clone()
    first = opt.step(f)
    assert torch.equal(f, keep)
    assert torch.equal(opt.step(f)[:2], first[:2])


def test_clip_takes_gradients_in_any_order_of_memory():
    """A parameter whose strides are not row-major has such a gradient; one set by hand may have gaps."""
    ps = params()
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(5, 40, generator=g, device="cuda")
    sum((p * p).float().sum() for p in ps).backward()
    (x @ ps[2]).sum().backward()
    assert not ps[2].grad.is_contiguous()
    ps[0].grad = torch.randn(20, 60, generator=g, device="cuda")[:, ::2]
    want, st = engine.clip_by_global_norm([p.grad for p in ps], 0.5)
    grads = [p.grad for p in ps]
    opt = train.ClippedOptimiser(torch.optim.SGD(ps, lr=0.1), 0.5)
    stats = opt.clip()
    # the sums of squares add up in memory's order: 64-bit sums, below 2^-40 apart, then one rounding to fp32
    assert bool(((stats - st).abs() <= 2.0 ** -23 * st).all())
    for p, g, w in zip(ps, grads, want):
        assert p.grad is g and p.grad.stride() == g.stride()
        assert bool(((g.float() - w.float()).abs() <= (2.0 ** -21 if g.dtype == torch.float32 else 2.0 ** -7) * w.float().abs()).all())
    norm = torch.sqrt(sum((g.double() ** 2).sum() for g in grads))
    assert abs(float(norm) - 0.5) <= 0.5 * 2.0 ** -8
    alone = train.ClippedOptimiser(torch.optim.SGD(ps, lr=0.1), None).clip()
    assert bool(((alone - engine.global_norm(grads)).abs() <= 2.0 ** -23 * alone).all())
