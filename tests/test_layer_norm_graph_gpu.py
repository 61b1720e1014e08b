"""Gradients of a layer norm's output taken after its gradient's own, on the GPU."""

import pytest
import torch

from fsctep_amd import learn_ops as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("shape", [(5, 20), (70, 640)])
def test_the_output_is_differentiated_after_its_gradient(shape, activation):
    """The same values as from a graph that was kept, to the bit."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x0, w0, dy, v, ey = (torch.randn(*s, generator=g, device="cuda") for s in (shape, shape[1:], shape, shape, shape))

    def grads(keep):
        x, w = x0.clone().requires_grad_(True), w0.clone().requires_grad_(True)
        y = L.layer_norm(x, w, None, activation=activation)
        dx, = torch.autograd.grad(y, x, dy, create_graph=True)
        gx, = torch.autograd.grad(dx, x, v, retain_graph=keep)
        return (gx, *torch.autograd.grad(y, (x, w), ey))

    assert all(torch.equal(a, b) for a, b in zip(grads(False), grads(True)))
