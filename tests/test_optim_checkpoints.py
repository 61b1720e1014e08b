"""Checkpoints that optim.AdamW takes and refuses, without a GPU: loading takes no step."""

import pytest
import torch

from fsctep_amd import optim


def stepped(kind, p=None, grad=None, **settings):
    """An optimiser of a kind with its states made by one step."""
    p = torch.linspace(-1, 1, 300).requires_grad_(True) if p is None else p
    opt = kind([p], **settings)
    p.grad = torch.ones_like(p) if grad is None else grad
    opt.step()
    return opt


def mine(dtype=torch.float32, n=300, **settings):
    return optim.AdamW([torch.zeros(n, dtype=dtype, requires_grad=True)], lr=0.25, **settings)


def refused(opt, state_dict, match):
    """Refused, with the optimiser as it was."""
    with pytest.raises(ValueError, match=match):
        opt.load_state_dict(state_dict)
    assert opt.param_groups[0]["lr"] == 0.25 and not opt.state


@pytest.mark.parametrize("kind,settings,match", [
    (torch.optim.Adam, dict(weight_decay=0.1), "decoupled"), (torch.optim.NAdam, dict(weight_decay=0.1), "another optimiser"),
    (torch.optim.NAdam, dict(), "another optimiser"), (torch.optim.NAdam, dict(decoupled_weight_decay=True), "another optimiser"),
    (torch.optim.RAdam, dict(weight_decay=0.1), "another optimiser"), (torch.optim.RAdam, dict(), "another optimiser"),
    (torch.optim.Adamax, dict(), "bits"), (torch.optim.AdamW, dict(amsgrad=True), "amsgrad")])
def test_checkpoints_of_other_rules_are_refused(kind, settings, match):
    """Their states have the same names, or some of them; stepped on by another rule they would be misread in silence."""
    refused(mine(), stepped(kind, lr=0.5, **settings).state_dict(), match)


def test_a_checkpoint_without_the_settings_is_refused():
    p = torch.zeros(3, requires_grad=True)
    theirs = stepped(torch.optim.SparseAdam, p, torch.ones(3).to_sparse())
    refused(mine(n=3), theirs.state_dict(), "another optimiser")


def test_a_checkpoint_with_other_states_is_refused():
    held = stepped(torch.optim.AdamW, lr=0.5).state_dict()
    held["state"][0]["momentum_buffer"] = torch.zeros(300)
    refused(mine(), held, "momentum_buffer")


@pytest.mark.parametrize("kind,settings", [(torch.optim.AdamW, dict(weight_decay=0.1)), (torch.optim.AdamW, dict(foreach=True)),
                                           (torch.optim.Adam, dict())])
def test_checkpoints_of_the_same_rule_are_taken(kind, settings):
    """Adam without a weight decay is AdamW without one."""
    theirs, opt = stepped(kind, lr=0.5, **settings), mine()
    opt.load_state_dict(theirs.state_dict())
    (a,), (b,) = theirs.state.values(), opt.state.values()
    assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["weight_decay"] == theirs.param_groups[0]["weight_decay"]
    assert all(torch.equal(a[k], b[k]) for k in ("step", "exp_avg", "exp_avg_sq")) and len(b) == 3
    # and from there on into one of this kind
    other = mine()
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["lr"] == 0.5


def test_a_checkpoint_of_a_scheduled_run_is_taken():
    """What schedulers leave in a group is no setting of a rule."""
    theirs = stepped(torch.optim.AdamW, lr=0.5)
    torch.optim.lr_scheduler.OneCycleLR(theirs, 1.0, total_steps=10)
    opt = mine()
    opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["lr"] == theirs.param_groups[0]["lr"]
