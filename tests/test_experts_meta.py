"""The expert readout's operators on Meta tensors: forward-mode derivatives and arguments that the GPU refuses are refused
there too."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from fsctep_amd import expert_ops as X
from test_experts_host import meta


def mlp_args(dtype=torch.float32):
    return dict(x=meta(7, 20, dtype=dtype), index=meta(7, 3, dtype=torch.int32), weight=meta(7, 3),
                w_in=meta(6, 18, 20, dtype=dtype), w_out=meta(6, 20, 9, dtype=dtype))


FORWARD_MODE = ([("norm", n) for n in ("x", "weight", "residual")] + [("route", "logits")] +
                [("mlp", n) for n in ("x", "weight", "w_in", "w_out")] + [("norm_q8", "x")])


@pytest.mark.parametrize("op,which", FORWARD_MODE)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(op, which, grad):
    """A tangent is not dropped, with and without grad mode."""
    args = dict(norm=dict(x=meta(7, 20), weight=meta(20), residual=meta(7, 20)), route=dict(logits=meta(7, 6), k=3),
                norm_q8=dict(x=meta(7, 20), weight=meta(20)), mlp=mlp_args())[op]
    call = dict(norm=X.rms_norm, norm_q8=X.rms_norm_q8, route=X.route_experts, mlp=X.expert_mlp)[op]
    with torch.set_grad_enabled(grad), fwd.dual_level():
        args[which] = fwd.make_dual(args[which], torch.empty_like(args[which]))
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward AD|Forward AD"):
            call(**args)
