"""The training step's energy head with modules whose call someone has taken over (offloading and quantisation libraries put a
forward of their own on a module), on the GPU."""

import pytest
import torch

from fsctep_amd import learn_ops, train_ops as T
from test_learn_trunk_gpu import DEV, head

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["norm", "net"])
def test_a_forward_put_on_a_module_is_called(monkeypatch, which):
    net, ws = head()
    x = torch.randn(7, 224, device=DEV)
    calls, own = [], []
    real = learn_ops.layer_norm
    monkeypatch.setattr(learn_ops, "layer_norm", lambda *a, **k: own.append(1) or real(*a, **k))
    T.readout_energy(net, ws, x)
    assert len(own) == 4
    own.clear()
    module = net if which == "net" else net.layer_norms[1]
    plain = module.forward
    module.forward = lambda t: calls.append(1) or 2 * plain(t)
    want = ws(net(x))
    calls.clear()
    assert torch.equal(T.readout_energy(net, ws, x), want) and calls and not own
    del module.forward
    T.readout_energy(net, ws, x)
    assert len(own) == 4
