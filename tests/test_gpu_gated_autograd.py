"""Gradients of the gated projection that autograd hands over in other places than a fresh tensor's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _leaves(dev):
    g = torch.Generator(device=dev).manual_seed(4)
    x, w, z = (torch.randn(s, generator=g, device=dev).bfloat16() for s in ((20, 72), (80, 72), (3 + 20 * 40,)))
    return x.requires_grad_(), w.requires_grad_(), z


@pytest.mark.parametrize("way", ["function", "operator", "compiled"])
def test_a_gradient_that_begins_between_16_byte_lines(et, dev, way):
    """h behind three other values of one vector: its gradient is a view from the fourth value on."""
    def f(x, w, z):
        h = et.gated_linear_autograd(x, w) if way == "function" else torch.ops.etmoe.gated_linear(x, w, "silu")
        return (torch.cat([z[:3], h.reshape(-1)]).float() * z.float()).sum()

    x, w, z = _leaves(dev)
    (torch.compile(f, fullgraph=True, backend="aot_eager") if way == "compiled" else f)(x, w, z).backward()
    dx, dw = et.gated_linear_backward(z[3:].view(20, 40).clone(), x.detach(), w.detach())
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)


def test_a_gradient_of_columns_and_of_a_transpose(et, dev):
    x, w, z = _leaves(dev)
    c = z[3:].view(20, 40)
    h = et.gated_linear_autograd(x, w)
    (h.t().float() * c.t().contiguous().float()).sum().backward()
    dx, dw = et.gated_linear_backward(c.clone(), x.detach(), w.detach())
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
    x.grad = w.grad = None
    wide = torch.cat([torch.zeros(20, 5, device=dev).bfloat16(), et.gated_linear_autograd(x, w)], 1)
    (wide[:, 5:].float() * c.float()).sum().backward()
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
