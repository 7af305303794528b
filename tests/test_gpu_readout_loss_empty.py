"""The read-out's cross-entropy over an empty batch, past the few-classes kernel."""
import pytest
import torch

from gncde import autograd, engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead,hidden,classes", [((0,), 64, 5000), ((0,), 333, 1001), ((3, 0, 2), 4096, 700)])
@pytest.mark.parametrize("kind", ["i64", "rows"])
def test_gradients_of_no_rows(lead, hidden, classes, dtype, kind):
    x = torch.zeros(*lead, hidden, dtype=dtype, device="cuda", requires_grad=True)
    W = torch.randn(classes, hidden, device="cuda").to(dtype).requires_grad_()
    b = torch.randn(classes, device="cuda").to(dtype).requires_grad_()
    y = torch.zeros(*lead, dtype=torch.int64, device="cuda") if kind == "i64" else \
        torch.zeros(*lead, classes, device="cuda")
    loss = autograd.linear_cross_entropy(x, W, b, y)
    assert loss.shape == lead
    loss.sum().backward()
    assert x.grad.shape == x.shape
    assert W.grad.shape == W.shape and b.grad.shape == b.shape
    assert bool((W.grad == 0).all()) and bool((b.grad == 0).all())
    _, stats = engine.linear_cross_entropy(x.detach(), W.detach(), b.detach(), y)
    g = torch.zeros(lead, device="cuda")
    gx, gW, gb = engine.linear_cross_entropy_grad(x.detach(), W.detach(), b.detach(), y, stats, g, None, True, False, True)
    assert gx.shape == x.shape and gW is None and bool((gb == 0).all())
