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
