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


def test_moments_of_16_bits_are_loaded_in_32():
    """torch.optim.AdamW holds the moments of a bfloat16 parameter in bfloat16."""
    p = torch.linspace(-1, 1, 300).bfloat16().requires_grad_(True)
    theirs, opt = stepped(torch.optim.AdamW, p, lr=0.5), mine(torch.bfloat16)
    opt.load_state_dict(theirs.state_dict())
    (a,), (b,) = theirs.state.values(), opt.state.values()
    for name in ("exp_avg", "exp_avg_sq"):
        assert a[name].dtype == torch.bfloat16 and b[name].dtype == torch.float32 and torch.equal(a[name].float(), b[name])


def state_of_8_bits(n=300):
    return dict(step=torch.ones(()), exp_avg=torch.zeros(n, dtype=torch.uint8), exp_avg_scale=torch.ones(2),
                root=torch.zeros(n, dtype=torch.uint8), root_scale=torch.ones(2))


@pytest.mark.parametrize("bits,change,match", [
    (32, dict(exp_avg=torch.zeros(299)), "exp_avg is"), (32, dict(exp_avg_sq=torch.zeros(300, 2)), "exp_avg_sq is"),
    (32, dict(step=torch.zeros(2)), "step is"), (32, dict(master=torch.zeros(3)), "master is"),
    (32, dict(exp_avg=torch.zeros(300, dtype=torch.uint8)), "exp_avg is"), (32, dict(step=None), "step count"),
    (8, dict(exp_avg=torch.zeros(300)), "exp_avg is"), (8, dict(root=torch.zeros(301, dtype=torch.uint8)), "root is"),
    (8, dict(root_scale=torch.ones(3)), "root_scale is"), (8, dict(exp_avg_scale=torch.ones(2, dtype=torch.uint8)), "scale is"),
    (8, dict(step=None), "step count")])
def test_states_of_other_sizes_and_types_are_refused(bits, change, match):
    """Before the optimiser's own states go."""
    held = stepped(torch.optim.AdamW, lr=0.5).state_dict()
    if bits == 8:
        held["state"][0] = state_of_8_bits()
    held["state"][0] = {k: v for k, v in (held["state"][0] | change).items() if v is not None}
    refused(mine(state_bits=bits), held, match)


def test_states_of_8_bits_are_loaded_apart_from_the_checkpoint():
    held = mine(state_bits=8).state_dict()
    held["state"][0] = state_of_8_bits()
    opt = mine(state_bits=8)
    opt.load_state_dict(held)
    (s,) = opt.state.values()
    for name, t in held["state"][0].items():
        assert torch.equal(s[name], t) and s[name].dtype == t.dtype and s[name].data_ptr() != t.data_ptr()


def test_states_of_any_order_are_loaded_contiguous():
    p = torch.zeros(20, 30, requires_grad=True)
    held = stepped(torch.optim.AdamW, torch.ones(20, 30, requires_grad=True), lr=0.5).state_dict()
    turned = torch.randn(30, 20).t()
    held["state"][0]["exp_avg"], held["state"][0]["step"] = turned, 7
    opt = optim.AdamW([p])
    opt.load_state_dict(held)
    assert torch.equal(opt.state[p]["exp_avg"], turned) and opt.state[p]["exp_avg"].is_contiguous()
    assert opt.state[p]["step"].shape == () and float(opt.state[p]["step"]) == 7


def test_a_copy_is_held_for_16_bit_parameters_alone():
    """A bfloat16 run's copies would stand still beside float32 parameters, and be taken for theirs when those go back."""
    held = stepped(torch.optim.AdamW, lr=0.5).state_dict()
    held["state"][0]["master"] = torch.full((300,), 5.0)
    for dtype, there in ((torch.float32, False), (torch.bfloat16, True)):
        opt = mine(dtype)
        opt.load_state_dict(held)
        (s,) = opt.state.values()
        assert ("master" in s) == there and ("master" in opt.state_dict()["state"][0]) == there
    del held["state"][0]["master"]
    opt = mine(torch.bfloat16)
    opt.load_state_dict(held)
    (s,) = opt.state.values()
    assert "master" not in s           # the parameter's values may still be to come; the first step copies them


def test_a_learning_rate_of_64_bits_is_loaded_in_32():
    held = stepped(torch.optim.AdamW, lr=torch.tensor(0.125, dtype=torch.float64), foreach=False).state_dict()
    opt = mine()
    opt.load_state_dict(held)
    assert opt.param_groups[0]["lr"].dtype == torch.float32 and float(opt.param_groups[0]["lr"]) == 0.125
