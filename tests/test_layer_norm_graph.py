"""What a run through the layer norm's autograd graph uses up, on Meta tensors (no values, no GPU)."""

import pytest
import torch

from fsctep_amd import learn_ops as L


def force(x, w, dy, norm):
    """y and its gradient, which can be differentiated again."""
    y = norm(x, w)
    return y, torch.autograd.grad(y, x, dy, create_graph=True)[0]


def leaves():
    return tuple(torch.empty(*s, device="meta", requires_grad=True) for s in ((7, 20), (20,), (7, 20)))


def own(x, w):
    return L.layer_norm(x, w, None)


def own_silu(x, w):
    return L.layer_norm(x, w, None, activation="silu")


def torchs(x, w):
    return torch.nn.functional.layer_norm(x, (20,), w)


@pytest.mark.parametrize("norm", [own, own_silu, torchs])
@pytest.mark.parametrize("later", ["x", "w", "both"])
def test_the_output_can_be_differentiated_after_its_gradient(norm, later):
    """The gradient of dx with respect to x passes through the norm's node without using it up, as it passes by torch's."""
    x, w, dy = leaves()
    y, dx = force(x, w, dy, norm)
    gx, = torch.autograd.grad(dx.sum(), x)
    ask = dict(x=[x], w=[w], both=[x, w])[later]
    got = torch.autograd.grad(y.sum(), ask)
    assert gx.shape == x.shape and [t.shape for t in got] == [t.shape for t in ask]


@pytest.mark.parametrize("norm", [own, own_silu, torchs])
def test_a_graph_that_was_used_up_says_so(norm):
    for twice in (lambda y, dx, x: y, lambda y, dx, x: dx):
        x, w, dy = leaves()
        end = twice(*force(x, w, dy, norm), x)
        torch.autograd.grad(end.sum(), x)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(end.sum(), x)
    # y and dx together use up both, in one run
    x, w, dy = leaves()
    y, dx = force(x, w, dy, norm)
    torch.autograd.grad(y.sum() + dx.sum(), x)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y.sum(), w)


def test_a_kept_graph_runs_as_often_as_asked():
    x, w, dy = leaves()
    y, dx = force(x, w, dy, own)
    for _ in range(2):
        torch.autograd.grad(dx.sum(), x, retain_graph=True)
        torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
        torch.autograd.grad(y.sum() + dx.sum(), (x, w), retain_graph=True)
    torch.autograd.grad(y.sum() + dx.sum(), (x, w))


def test_a_graph_of_gradients_only_passed_on_is_let_go():
    """Nothing of a dropped graph is kept alive by a run that used nothing up."""
    import gc
    import weakref
    x, w, dy = leaves()
    h = x * 1.0
    y, dx = force(h, w, dy, own)
    torch.autograd.grad(dx.sum(), h)
    ref = weakref.ref(h)
    del h, y, dx
    gc.collect()
    assert ref() is None
