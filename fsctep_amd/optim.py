"""AdamW on the GPU: two launches for each 48 tensors, the gradients clipped by their common norm on the way (one launch
for each 48 tensors more, and one), states in 32 or in 8 bits.

    opt = AdamW(model.parameters(), lr=1e-3, weight_decay=0.01, max_norm=1.0)       # a torch.optim.Optimizer
    loss.backward(); opt.step(); opt.zero_grad()
    opt.grad_norm                                                                    # of the last step, on the GPU

The formulas are torch.optim.AdamW's (the reference's trainer, training/trainer.py), states of 32 bits have its names,
so that its checkpoints load (other optimisers' are refused).  Parameters are float32, or bfloat16 with a float32 copy
("master") in the state that is stepped and rounded (who writes other values into such a parameter writes them into its
copy as well).  Step counts live on the GPU and nothing waits for it, so a step can be captured into a graph (``lr`` as a
float32 tensor then changes between replays).  The ops are registered in C++ (``csrc/torch_learn_ops.cpp``, kernels
``csrc/adamw.hip``).

States in 8 bits (``state_bits=8``): m and sqrt(v) as 8-bit floats with a float32 scale for each 256 values, rounded
up or down by a hash of the value's number and the step, so that small changes add up over the steps instead of being
rounded away.  16 bytes a value are moved in place of 28.  The format reaches down to 2e-5 of the largest of the 256: a value
whose gradients stay below that share of its neighbours' loses its momentum (m becomes 0), and its steps are divided by
the smallest sqrt(v) there is, which makes them smaller than its own would.

    train_step(model, optimizer, pos, batch, cell, graph, energy, forces, ...)       # a trunk's step on energies and forces
    adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, lr, betas, eps, weight_decay, max_norm, masters, norm)
    adamw_step_q8(params, grads, exp_avgs, exp_avg_scales, roots, root_scales, steps, ...)
    grad_norm(grads) -> norm
    moment_values(codes, scale), root_values(codes, scale) -> what 8-bit states stand for
"""

from __future__ import annotations

from . import _lib

_lib.load_torch_ops()

import math  # noqa: E402

import torch  # noqa: E402

GROUP = 256            # values that share a scale


@torch.no_grad()
def grad_norm(grads):
    """The 2-norm of all values of the gradients (float32 or bfloat16), a float32 on the GPU; sums in 64 bits."""
    grads = list(grads)
    if not grads:
        raise ValueError("grad_norm: no gradients")
    return torch.ops.fsctep.grad_norm(grads)


def _settings(grads, lr, betas, eps, weight_decay, max_norm, norm):
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError(f"betas must lie in [0, 1), got {betas}")
    if eps < 0 or weight_decay < 0 or (not isinstance(lr, torch.Tensor) and lr < 0):
        raise ValueError("lr, eps and weight_decay must not be negative")
    if max_norm is not None and not max_norm > 0:
        raise ValueError(f"max_norm must be positive, got {max_norm}")
    if max_norm is None:
        norm = None
    elif norm is None and len(grads):
        norm = torch.ops.fsctep.grad_norm(grads)
    t = lr if isinstance(lr, torch.Tensor) else None
    return norm, (norm, t, 0.0 if t is not None else float(lr), float(betas[0]), float(betas[1]), float(eps),
                  float(weight_decay), 0.0 if max_norm is None else float(max_norm))


@torch.no_grad()
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, max_norm: float | None = None, masters=None, norm=None):
    """One AdamW step in place on lists of contiguous tensors: ``params`` float32 or bfloat16, ``grads`` of their types,
    moments float32, ``steps`` one float32 value each on the GPU (the steps taken before), ``masters`` float32 copies
    where a parameter is bfloat16.  ``lr``: a number or one float32 value on the GPU.  ``max_norm``: the gradients
    count as scaled by min(1, max_norm / (norm + 1e-6)), ``norm`` their norm where the caller has it (of more tensors,
    say).  Returns the norm (None without ``max_norm``)."""
    grads = list(grads)
    norm, rest = _settings(grads, lr, betas, eps, weight_decay, max_norm, norm)
    lists = [list(t) for t in (params, grads, exp_avgs, exp_avg_sqs, steps, masters or [])]
    if any(lists):
        torch.ops.fsctep.adamw_(*lists, *rest)
    return norm


@torch.no_grad()
def adamw_step_q8(params, grads, exp_avgs, exp_avg_scales, roots, root_scales, steps, lr=1e-3, betas=(0.9, 0.999),
                  eps: float = 1e-8, weight_decay: float = 1e-2, max_norm: float | None = None, masters=None, norm=None):
    """``adamw_step`` with states in 8 bits: codes (uint8, as many as values) and scales (float32, one for each 256) of
    the first moment and of the second moment's root; all zeros at the start."""
    grads = list(grads)
    norm, rest = _settings(grads, lr, betas, eps, weight_decay, max_norm, norm)
    lists = [list(t) for t in (params, grads, exp_avgs, exp_avg_scales, roots, root_scales, steps, masters or [])]
    if any(lists):
        torch.ops.fsctep.adamw_q8_(*lists, *rest)
    return norm


def moment_values(codes, scale):
    """The first moments that 8-bit codes stand for, float32."""
    return torch.ops.fsctep.adamw_values(codes, scale, False)


def root_values(codes, scale):
    """The second moments' roots that 8-bit codes stand for, float32."""
    return torch.ops.fsctep.adamw_values(codes, scale, True)


def _check_rule(group):
    """Refuses a checkpoint's group whose settings are not of AdamW without its variants."""
    for name in ("amsgrad", "maximize"):
        if group.get(name):
            raise ValueError(f"the checkpoint is of an optimiser with {name}, which this one does not have")
    missing = {"lr", "betas", "eps", "weight_decay"} - set(group)
    # torch's Adam and AdamW always say amsgrad; NAdam and RAdam, whose states have the same names, never do
    if missing or "momentum_decay" in group or ("maximize" in group and "amsgrad" not in group):
        raise ValueError(f"the checkpoint is of another optimiser: its settings are {sorted(set(group) - {'params'})}")
    if group.get("decoupled_weight_decay") is False and group["weight_decay"] != 0:
        raise ValueError("the checkpoint is of an optimiser whose weight_decay is not decoupled from the gradient (Adam)")


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` without its variants, on the GPU, for float32 and bfloat16 parameters (contiguous).
    ``max_norm`` clips by the norm of all groups' gradients together (``grad_norm`` holds the last one's; a norm that is
    not finite makes the step what the formulas say, NaN and all).  ``state_bits``: 32 or 8."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 max_norm: float | None = None, state_bits: int = 32):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        _settings([], lr, betas, eps, weight_decay, max_norm, None)
        self.max_norm, self.state_bits, self.grad_norm = max_norm, int(state_bits), None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        return super().__getstate__() | {"max_norm": self.max_norm, "state_bits": self.state_bits, "grad_norm": None}

    def _state(self, p):
        s = self.state[p]
        copied = p.dtype == torch.bfloat16
        if (not s or (copied and "master" not in s)) and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: take a step before one is captured (a replay would start the states anew)")
        if not s:
            s["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            if self.state_bits == 32:
                for name in ("exp_avg", "exp_avg_sq"):
                    s[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            else:
                for name in ("exp_avg", "root"):
                    s[name] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
                    s[name + "_scale"] = torch.zeros(math.ceil(p.numel() / GROUP), dtype=torch.float32, device=p.device)
        if copied and "master" not in s:     # a checkpoint without copies: of what the parameter holds now
            s["master"] = p.detach().float()
        if not copied:                       # the model went from bfloat16 to float32
            s.pop("master", None)
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = [(g, [p for p in g["params"] if p.grad is not None]) for g in self.param_groups]
        if self.max_norm is not None:
            grads = [p.grad for _, ps in groups for p in ps]
            self.grad_norm = grad_norm(grads) if grads else None
        names = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("exp_avg", "exp_avg_scale", "root", "root_scale")
        call = adamw_step if self.state_bits == 32 else adamw_step_q8
        for g, ps in groups:
            if not ps:
                continue
            states = [self._state(p) for p in ps]
            call(ps, [p.grad for p in ps], *([s[n] for s in states] for n in names), [s["step"] for s in states],
                 lr=g["lr"], betas=g["betas"], eps=g["eps"], weight_decay=g["weight_decay"], max_norm=self.max_norm,
                 masters=[s.get("master", p) for s, p in zip(states, ps)], norm=self.grad_norm)
        return loss

    def _loaded(self, p, held):
        """A parameter's state from a checkpoint's, in this optimiser's types (torch's moments have their parameter's)."""
        codes, values, scales = (torch.uint8, p.shape), (torch.float32, p.shape), (torch.float32, (math.ceil(p.numel() / GROUP),))
        kinds = dict(step=(torch.float32, ()), exp_avg=values if self.state_bits == 32 else codes, exp_avg_sq=values, root=codes,
                     exp_avg_scale=scales, root_scale=scales, master=values)
        out = {}
        for name, value in held.items():
            dtype, shape = kinds[name]
            value = torch.as_tensor(value)
            if value.numel() != math.prod(shape) or (value.dtype == torch.uint8) != (dtype == torch.uint8):
                raise ValueError(f"the checkpoint's {name} is {tuple(value.shape)} of {value.dtype}, its parameter {tuple(p.shape)}")
            out[name] = value.detach().to(p.device, dtype, copy=True).reshape(shape).contiguous()
        if p.dtype != torch.bfloat16:
            out.pop("master", None)          # of a bfloat16 run: no step would keep it up
        return out

    def load_state_dict(self, state_dict):
        """Also a checkpoint of ``torch.optim.AdamW`` without its variants (states in 32 bits).  States keep their own types,
        which the base class would cast to the parameter's.  What is refused is refused before anything changes."""
        held = state_dict["state"]
        want = {"exp_avg", "exp_avg_sq"} if self.state_bits == 32 else {"exp_avg", "exp_avg_scale", "root", "root_scale"}
        if not all(want <= set(s) for s in held.values() if s):
            raise ValueError(f"the checkpoint's states do not have {self.state_bits} bits")
        for g in state_dict["param_groups"]:
            _check_rule(g)
        for s in held.values():
            if s and set(s) - want - {"step", "master"}:
                raise ValueError(f"the checkpoint is of another optimiser: it has states "
                                 f"{sorted(set(s) - want - {'step', 'master'})}")
            if s and "step" not in s:
                raise ValueError("the checkpoint has a state without its step count")
        ready = {}
        for mine, theirs in zip(self.param_groups, state_dict["param_groups"]):
            ready.update((p, self._loaded(p, held[i])) for p, i in zip(mine["params"], theirs["params"]) if held.get(i))
        super().load_state_dict(state_dict)
        self.state.update(ready)
        for g in self.param_groups:          # a checkpoint read to the host, or one of 64 bits
            if isinstance(g["lr"], torch.Tensor) and g["params"]:
                g["lr"] = g["lr"].detach().to(g["params"][0].device, torch.float32)


def train_step(model, optimizer, pos, batch, cell, graph, energy, forces, energy_weight: float = 1.0,
               force_weight: float = 1.0, external_tensor=None):
    """One training step of a trunk in ``train()`` mode on a prepared graph (``sparse.energy_and_forces`` and
    ``ictd.energy_forces`` are the same evaluation without the step): energies (G,) of the structures and forces F = -dE/dpos
    (N, 3), loss = energy_weight mean (E - energy)^2 + force_weight mean (F - forces)^2 (training/trainer.py:1292-1297),
    its gradients, and the optimiser's step.  Returns (loss, E, F), detached; nothing waits for the GPU."""
    if not model.training:
        raise ValueError("train_step: the model is not in train() mode")
    if tuple(energy.shape) != (cell.shape[0],) or forces.shape != pos.shape:
        raise ValueError(f"train_step: energy must be ({cell.shape[0]},) and forces {tuple(pos.shape)}, "
                         f"got {tuple(energy.shape)} and {tuple(forces.shape)}")
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        # torch's sums over many blocks clear memory by nodes that a replay does not repeat reliably
        raise RuntimeError("train_step is not captured into a graph; the optimiser's step by itself can be")
    optimizer.zero_grad(set_to_none=True)
    pos = pos.detach().requires_grad_(True)
    if external_tensor is None:
        out = model.forward_graph(pos, batch, cell, graph)
    else:
        out = model.forward_graph(pos, batch, cell, graph, external_tensor=external_tensor)
    atoms = (out[0] if isinstance(out, tuple) else out).squeeze(-1)
    # the sum by structure is the gradient of a lookup of each atom's structure
    total = torch.ops.fsctep.embedding_backward(atoms.unsqueeze(1), batch, cell.shape[0], 1.0).squeeze(1)
    gradient, = torch.autograd.grad(atoms.sum(), pos, create_graph=True)
    loss = (energy_weight * (total - energy).square().mean()
            + force_weight * (gradient + forces).square().mean())
    # of the parameters alone: the positions are not trained
    params = [p for group in optimizer.param_groups for p in group["params"] if p.requires_grad]
    for p, g in zip(params, torch.autograd.grad(loss, params, allow_unused=True)):
        p.grad = g
    optimizer.step()
    return loss.detach(), total.detach(), -gradient.detach()
