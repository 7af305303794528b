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


def loss_terms(ps, x):
    """A sum of squares over parameters of both types, and its element count on the device; the last one takes no part."""
    y = (x @ ps[0])[:, :8].to(torch.bfloat16) @ ps[1]
    return (y.float() ** 2).sum() + ((x[:, :1] * ps[2].sum(0)) ** 2).sum(), torch.tensor(5 * 7, device="cuda")


@pytest.mark.parametrize("kind", ["sgd", "adamw"])
@pytest.mark.parametrize("max_norm", [0.05, 1e4, None])
def test_make_step_clips_gradients_as_they_lie(kind, max_norm, monkeypatch):
    """One process: the mean loss's gradients reach the clip in the parameters' own tensors, with no flat copy on the way; a
    parameter without one counts as zeros (weight decay applies to it), as in the flat gradient."""
    make = {"sgd": lambda ps: torch.optim.SGD(ps, lr=0.1), "adamw": lambda ps: torch.optim.AdamW(ps, lr=0.1, weight_decay=0.1)}
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(5, 20, generator=g, device="cuda")
    a, b = params(), params()
    opt = train.ClippedOptimiser(make[kind](a), max_norm)
    monkeypatch.setattr(opt, "flat_grad", lambda: pytest.fail("a flat gradient"))
    got = train.make_step(opt, loss_terms, a, x)

    sse, count = loss_terms(b, x)
    (sse / count).backward()
    for p in b:
        p.grad = torch.zeros_like(p) if p.grad is None else p.grad
    stats = train.ClippedOptimiser(make[kind](b), max_norm).clip()
    before = [p.detach().clone() for p in b]
    make[kind](b).step()
    for p, q in zip(a, b):
        assert torch.equal(p, q) and torch.equal(p.grad, q.grad) and p.grad.stride() == q.grad.stride()
    assert abs(float(got[0]) - float(sse.detach()) / 35) <= 2.0 ** -22 * abs(float(got[0]))
    assert torch.equal(got[1], stats[1])
    assert float(got[2]) == max(float((p.detach() - z).abs().max()) for p, z in zip(b, before))
    if kind == "adamw":
        assert not torch.equal(a[3], params()[3])


@pytest.mark.parametrize("max_norm", [0.05, None])
def test_make_step_of_several_ranks_reduces_one_flat_gradient(max_norm, monkeypatch):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(5, 20, generator=g, device="cuda")
    a, b = params(), params()
    monkeypatch.setattr(train, "dist_world", lambda: (0, 2))
    got = train.make_step(train.ClippedOptimiser(torch.optim.SGD(a, lr=0.1), max_norm), loss_terms, a, x)
    ref = train.ClippedOptimiser(torch.optim.SGD(b, lr=0.1), max_norm)
    sse, count = loss_terms(b, x)
    sse.backward()
    mean, loss = train.reduce_gradients(ref.flat_grad(), sse, count)
    stats = ref.step(mean)
    assert all(torch.equal(p, q) and torch.equal(p.grad, q.grad) for p, q in zip(a, b))
    assert torch.equal(got[0], loss) and torch.equal(got[1], stats[1]) and torch.equal(got[2], stats[2])
