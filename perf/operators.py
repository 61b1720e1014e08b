"""The expert readout's operators: what a program hands to them, their plain forms, and the same in 64 bits.

Three operators on per-atom rows: a root-mean-square norm with the residual's addition (its output in the rows'
type or in 8 bits with a scale for each row), the router (scores, balance bias, groups, top-k, renormalised
weights), and the experts' gated products (16 or 32 bits with gradients, or 8-bit rows and weights).

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes what a
program holds before the call, ``run(state)`` is one pass, ``work(case)`` what the pass cannot do without and
``exact(case, seed)`` the outputs in 64 bits.  ``own`` selects between the plain form and the framework's calls.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
GROUP = 128            # hidden columns that share a scale in the 8-bit products
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # ---- norm
        # the step of a 32-atom molecule: one launch, latency
        {"name": "norm_32x640", "kind": "norm", "rows": 32, "width": 640, "dtype": "fp32", "residual": True,
         "form": "forward"},
        # training on the invariants of a large batch, forward and backward through both outputs
        {"name": "norm_train_100000x640", "kind": "norm", "rows": 100000, "width": 640, "dtype": "bf16",
         "residual": True, "form": "grad"},
        # screening: the wide (1600) invariants of a 10,007-atom system, to 8 bits for the products below
        {"name": "norm_q8_10007x1600", "kind": "norm", "rows": 10007, "width": 1600, "dtype": "bf16",
         "residual": True, "form": "q8"},
        # ---- router
        # the step of a 32-atom molecule
        {"name": "route_32x8", "kind": "route", "rows": 32, "experts": 8, "k": 2, "score": "softmax", "bias": False,
         "groups": 1, "kept": 1, "best": 1, "renormalise": True, "dtype": "fp32", "grad": False},
        # training: many experts in groups, balanced by a bias, with the logits' gradient
        {"name": "route_train_100000x256", "kind": "route", "rows": 100000, "experts": 256, "k": 8,
         "score": "sigmoid", "bias": True, "groups": 8, "kept": 4, "best": 2, "renormalise": True, "dtype": "fp32",
         "grad": True},
        # ---- experts' products
        # one row (one atom changed in a Monte Carlo move): the weights of its experts are read once
        {"name": "experts_1x640", "kind": "experts", "rows": 1, "width": 640, "hidden": 640, "experts": 8, "k": 2,
         "dtype": "fp32", "grads": "none"},
        # energy and forces of a 32-atom molecule: forward and the rows' gradient
        {"name": "experts_step_32x640", "kind": "experts", "rows": 32, "width": 640, "hidden": 640, "experts": 8,
         "k": 2, "dtype": "fp32", "grads": "rows"},
        # energy and forces at the headline size
        {"name": "experts_step_10000x640", "kind": "experts", "rows": 10000, "width": 640, "hidden": 640,
         "experts": 8, "k": 2, "dtype": "fp32", "grads": "rows"},
        # a training step on wide invariants in bf16, to all gradients
        {"name": "experts_train_16384x1600", "kind": "experts", "rows": 16384, "width": 1600, "hidden": 800,
         "experts": 16, "k": 2, "dtype": "bf16", "grads": "all"},
        # a training step at sizes that no tile divides
        {"name": "experts_train_4099x331", "kind": "experts", "rows": 4099, "width": 331, "hidden": 203,
         "experts": 5, "k": 2, "dtype": "fp32", "grads": "all"},
        # screening in 8 bits: energies of one molecule
        {"name": "experts_q8_32x640", "kind": "experts_q8", "rows": 32, "width": 640, "hidden": 640, "experts": 8,
         "k": 2},
        # screening in 8 bits: energies of a large batch
        {"name": "experts_q8_50000x640", "kind": "experts_q8", "rows": 50000, "width": 640, "hidden": 1280,
         "experts": 16, "k": 2},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "route", "experts", "experts", "experts_q8"])
    if kind == "norm":
        width = _log(rng, 16, 2048)
        rows = _log(rng, 1, min(100000, 64000000 // width))
        return {"kind": kind, "rows": rows, "width": width, "dtype": rng.choice(["fp32", "bf16"]),
                "residual": rng.random() < 0.7, "form": rng.choice(["forward", "grad", "q8"])}
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, 4, 256 // groups)
        kept = rng.randint(1, groups)
        return {"kind": kind, "rows": _log(rng, 1, 100000), "experts": experts, "groups": groups, "kept": kept,
                "best": rng.randint(1, 2), "k": rng.randint(1, min(8, kept * (experts // groups))),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5,
                "renormalise": rng.random() < 0.7, "dtype": rng.choice(["fp32", "bf16"]), "grad": rng.random() < 0.5}
    experts = _log(rng, 2, 32)
    c = {"kind": kind, "rows": 0, "width": _log(rng, 32, 1600), "hidden": _log(rng, 32, 1280), "experts": experts,
         "k": rng.randint(1, min(4, experts))}
    if kind == "experts":
        c |= {"dtype": rng.choice(["fp32", "bf16"]), "grads": rng.choice(["none", "rows", "all"])}
    most = 1.5e11 / (6.0 * c["width"] * c["hidden"] * c["k"])
    c["rows"] = _log(rng, 1, max(2, min(50000, int(most))))
    return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _routing(g, rows, experts, k):
    """Choices as a trained router makes them: some experts are chosen more often than others, no expert twice in a
    row, 1 row in 32 (padding of a batch) with none."""
    pull = _randn(g, rows, experts) + 0.5 * _randn(g, 1, experts)
    top, index = torch.sort(pull, dim=1, descending=True)
    weight = torch.softmax(top[:, :k], dim=1)
    none = torch.rand(rows, 1, generator=g, device=DEV) < (1 / 32 if rows > 1 else 0)
    return torch.where(none, -1, index[:, :k]).int().contiguous(), torch.where(none, 0.0, weight).contiguous()


def _to_8_bits(w):
    """8-bit codes with a scale for each row of the last dimension."""
    scale = w.abs().amax(-1) / 127
    return torch.round(w / scale.unsqueeze(-1)).to(torch.int8), scale


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    kind = case["kind"]
    if kind == "norm":
        t, h, dt = case["rows"], case["width"], DTYPES[case["dtype"]]
        # rows of different sizes, as the invariants of different species are
        size = torch.exp(0.5 * _randn(g, t, 1))
        s["x"] = (size * _randn(g, t, h)).to(dt)
        s["weight"] = (1 + 0.2 * _randn(g, h)).to(dt)
        s["residual"] = (size * _randn(g, t, h)).to(dt) if case["residual"] else None
        if case["form"] == "grad":
            s["dy"], s["dz"] = _randn(g, t, h).to(dt), _randn(g, t, h).to(dt)
            for name in ("x", "weight") + (("residual",) if case["residual"] else ()):
                s[name].requires_grad_(True)
    elif kind == "route":
        t, e = case["rows"], case["experts"]
        logits = _randn(g, t, e) + 0.5 * _randn(g, 1, e)
        # padded rows have no expert, and some rows (their species) may not use some experts
        barred = torch.rand(t, e, generator=g, device=DEV) < 0.02
        if t > 1:
            barred |= torch.rand(t, 1, generator=g, device=DEV) < 1 / 64
        s["logits"] = logits.masked_fill(barred, -math.inf).to(DTYPES[case["dtype"]])
        # the bias of a balancing rule that adds or takes 0.001 a step
        s["bias"] = 0.001 * torch.round(20 * _randn(g, e)) if case["bias"] else None
        if case["grad"]:
            s["logits"].requires_grad_(True)
            s["dweight"] = _randn(g, t, case["k"])
    else:
        t, h, f, e = case["rows"], case["width"], case["hidden"], case["experts"]
        x = _randn(g, t, h)
        w_in, w_out = _randn(g, e, 2 * f, h) / math.sqrt(h), _randn(g, e, h, f) / math.sqrt(f)
        s["index"], s["weight"] = _routing(g, t, e, case["k"])
        if kind == "experts_q8":
            s["x"], s["x_scale"] = _to_8_bits(x)
            s["w_in"], s["w_in_scale"] = _to_8_bits(w_in)
            s["w_out"], s["w_out_scale"] = _to_8_bits(w_out)
        else:
            dt = DTYPES[case["dtype"]]
            s["x"], s["w_in"], s["w_out"] = x.to(dt), w_in.to(dt), w_out.to(dt)
            if case["grads"] != "none":
                s["dy"] = _randn(g, t, h).to(dt)
                s["x"].requires_grad_(True)
            if case["grads"] == "all":
                for name in ("weight", "w_in", "w_out"):
                    s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------ plain forms
def _plain_norm(s):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x if s["residual"] is None else (x + s["residual"].float()).to(dt).float()
    # the mean square in 64 bits and its root rounded once, so that no 8-bit code hangs on the order of a sum
    rstd = (1 / torch.sqrt(z.double().square().mean(-1, keepdim=True) + EPS)).float()
    zn = z * rstd
    y = zn * w
    if s["form"] == "q8":
        most = y.abs().amax(-1, keepdim=True)
        scale = most / 127
        code = torch.where(most > 0, torch.round(y * torch.div(torch.full_like(most, 127.0), most)), 0.0)
        return {"y": code * scale, "z": z.to(dt)}
    out = {"y": y.to(dt), "z": z.to(dt)}
    if s["form"] == "grad":
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - zn * (g * zn).mean(-1, keepdim=True))
        if s["residual"] is not None:
            dx = dx + s["dz"].float()
        out |= {"dx": dx.to(dt), "dweight": (dy * zn).sum(0).to(dt)}
    return out


def _plain_route(s):
    l = s["logits"].float()
    t, e = l.shape
    if s["score"] == "softmax":
        m = l.amax(-1, keepdim=True)
        ex = torch.exp(l - torch.where(m > -math.inf, m, 0.0))
        total = ex.sum(-1, keepdim=True, dtype=torch.float64).float()  # no choice hangs on the order of this sum
        sc = ex / torch.where(total > 0, total, 1.0)
    else:
        sc = 1.0 / (1.0 + torch.exp(-l))
    c = sc if s["bias"] is None else sc + s["bias"]
    c = torch.where(l > -math.inf, c, -math.inf)
    n = s["groups"]
    if n > 1:
        top = torch.sort(c.view(t, n, e // n), dim=-1, descending=True)[0][..., : s["best"]]
        rank = torch.where(top > -math.inf, top, 0.0).sum(-1)
        rank = torch.where(top[..., 0] > -math.inf, rank, -math.inf)
        first = torch.sort(rank, dim=-1, descending=True, stable=True)[1][:, : s["kept"]]
        kept = torch.zeros(t, n, dtype=torch.bool, device=l.device).scatter_(1, first, True)
        c = torch.where(kept.repeat_interleave(e // n, 1), c, -math.inf)
    order = torch.sort(c, dim=-1, descending=True, stable=True)
    value, index = order[0][:, : s["k"]], order[1][:, : s["k"]]
    there = value > -math.inf
    picked = torch.where(there, sc.gather(1, index), 0.0)
    total = picked.sum(-1, keepdim=True) if s["renormalise"] else torch.ones_like(picked[:, :1])
    over = torch.where(total > 0, 1 / total, 0.0)
    weight = picked * over
    out = {"index": torch.where(there, index, -1).int(), "weight": weight}
    if s["grad"]:
        u = s["dweight"]
        d = u * over
        if s["renormalise"]:
            d = (u - (u * weight).sum(-1, keepdim=True)) * over
        d = torch.where(there, d, 0.0)
        if s["score"] == "softmax":
            dl = torch.zeros_like(l).scatter_(1, index, d * picked) - sc * (d * picked).sum(-1, keepdim=True)
        else:
            dl = torch.zeros_like(l).scatter_(1, index, d * picked * (1 - picked))
        out["dlogits"] = dl.to(s["logits"].dtype)
    return out


def _places(s):
    """Rows by expert: batches of one expert each, padded to the longest.  Few rows take a copy of their expert's
    weights each instead.  Returns (the batch's expert, or None for all in order; batch size; rows a batch; the
    place of each slot, the last one for slots with no expert)."""
    e = s["experts"]
    flat = s["index"].reshape(-1).long()
    there = flat >= 0
    if flat.numel() <= e:
        place = torch.where(there, torch.arange(flat.numel(), device=flat.device), flat.numel())
        return flat.clamp(min=0), flat.numel(), 1, place
    key = torch.where(there, flat, e)
    counts = torch.bincount(key, minlength=e + 1)[:e]
    most = max(int(counts.max()), 1)
    order = torch.sort(key, stable=True)[1]
    start = torch.cumsum(counts, 0) - counts
    sorted_key = key[order].clamp(max=e - 1)
    at = torch.empty_like(flat)
    at[order] = sorted_key * most + torch.arange(flat.numel(), device=flat.device) - start[sorted_key]
    return None, e, most, torch.where(there, at, e * most)


def _spread(rows, place, batches, most):
    """(batches, most, width) of the slots' rows, zeros where there is none."""
    buf = rows.new_zeros(batches * most + 1, rows.shape[1])
    buf[place] = rows
    return buf[:-1].view(batches, most, -1)


def _collect(batch, place):
    rows = batch.reshape(-1, batch.shape[-1])
    return torch.cat([rows, rows.new_zeros(1, rows.shape[1])])[place]


def _plain_experts(s):
    dt, k = s["x"].dtype, s["k"]
    which, batches, most, place = _places(s)
    w_in = s["w_in"].float() if which is None else s["w_in"][which].float()
    w_out = s["w_out"].float() if which is None else s["w_out"][which].float()
    f = s["hidden"]
    x = s["x"].float().repeat_interleave(k, 0)
    xb = _spread(x, place, batches, most)
    a = torch.bmm(xb, w_in.transpose(1, 2))
    gate, up = a[..., :f], a[..., f:]
    sig = 1 / (1 + torch.exp(-gate))
    act = gate * sig
    h = act * up
    o = _collect(torch.bmm(h, w_out.transpose(1, 2)), place)
    weight = s["weight"].reshape(-1, 1)
    out = {"y": (o * weight).view(-1, k, o.shape[1]).sum(1).to(dt)}
    if s["grads"] == "none":
        return out
    dyb = _spread(s["dy"].float().repeat_interleave(k, 0), place, batches, most)
    wb = _spread(weight, place, batches, most)
    p = torch.bmm(dyb, w_out)
    dh = p * wb
    da = torch.cat([dh * up * sig * (1 + gate * (1 - sig)), dh * act], -1)
    dx = _collect(torch.bmm(da, w_in), place)
    out["dx"] = dx.view(-1, k, dx.shape[1]).sum(1).to(dt)
    if s["grads"] == "all":
        out["dweight"] = _collect((p * h).sum(-1, keepdim=True), place).view(-1, k)
        dw_in, dw_out = torch.bmm(da.transpose(1, 2), xb), torch.bmm(dyb.transpose(1, 2), h * wb)
        if which is not None:
            dw_in = torch.zeros_like(s["w_in"], dtype=torch.float32).index_add_(0, which, dw_in)
            dw_out = torch.zeros_like(s["w_out"], dtype=torch.float32).index_add_(0, which, dw_out)
        out |= {"dw_in": dw_in.to(dt), "dw_out": dw_out.to(dt)}
    return out


def _plain_experts_q8(s):
    k, f = s["k"], s["hidden"]
    which, batches, most, place = _places(s)
    take = (lambda v: v) if which is None else (lambda v: v[which])
    w_in = take(s["w_in"]) * take(s["w_in_scale"]).unsqueeze(-1)
    w_out = take(s["w_out"]) * take(s["w_out_scale"]).unsqueeze(-1)
    x = (s["x"] * s["x_scale"].unsqueeze(-1)).repeat_interleave(k, 0)
    a = torch.bmm(_spread(x, place, batches, most), w_in.transpose(1, 2))
    h = a[..., :f] / (1 + torch.exp(-a[..., :f])) * a[..., f:]
    pad = -f % GROUP
    hg = torch.nn.functional.pad(h, (0, pad)).view(batches, most, -1, GROUP)
    top = hg.abs().amax(-1, keepdim=True)
    code = torch.where(top > 0, torch.round(hg * torch.div(torch.full_like(top, 127.0), top)), 0.0)
    h = (code * (top / 127)).view(batches, most, -1)[..., :f]
    o = _collect(torch.bmm(h, w_out.transpose(1, 2)), place) * s["weight"].reshape(-1, 1)
    return {"y": o.view(-1, k, o.shape[1]).sum(1).to(torch.bfloat16)}


# ------------------------------------------------------------------ the framework's calls
def _own_norm(s):
    from fsctep_amd import expert_ops as X
    if s["form"] == "q8":
        code, scale, z = X.rms_norm_q8(s["x"], s["weight"], s["residual"], EPS)
        return {"y": code * scale.unsqueeze(-1), "z": z}
    y, z = X.rms_norm(s["x"], s["weight"], s["residual"], EPS)
    out = {"y": y, "z": z}
    if s["form"] == "grad":
        if s["residual"] is None:
            dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
        else:
            dx, dw = torch.autograd.grad((y, z), (s["x"], s["weight"]), (s["dy"], s["dz"]))
        out |= {"dx": dx, "dweight": dw}
    return out


def _own_route(s):
    from fsctep_amd import expert_ops as X
    index, weight = X.route_experts(s["logits"], s["k"], score=s["score"], bias=s["bias"], groups=s["groups"],
                                    groups_kept=s["kept"], group_best=s["best"], renormalise=s["renormalise"])
    out = {"index": index, "weight": weight}
    if s["grad"]:
        out["dlogits"], = torch.autograd.grad(weight, s["logits"], s["dweight"])
    return out


def _own_experts(s):
    from fsctep_amd import expert_ops as X
    y = X.expert_mlp(s["x"], s["index"], s["weight"], s["w_in"], s["w_out"])
    if s["grads"] == "none":
        return {"y": y}
    if s["grads"] == "rows":
        return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    dx, dweight, dw_in, dw_out = torch.autograd.grad(y, (s["x"], s["weight"], s["w_in"], s["w_out"]), s["dy"])
    return {"y": y, "dx": dx, "dweight": dweight, "dw_in": dw_in, "dw_out": dw_out}


def _own_experts_q8(s):
    from fsctep_amd import expert_ops as X
    return {"y": X.expert_mlp_q8(s["x"], s["x_scale"], s["index"], s["weight"], s["w_in"], s["w_in_scale"],
                                 s["w_out"], s["w_out_scale"])}


def run(state):
    if own:
        return {"norm": _own_norm, "route": _own_route, "experts": _own_experts,
                "experts_q8": _own_experts_q8}[state["kind"]](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "route": _plain_route, "experts": _plain_experts,
                "experts_q8": _plain_experts_q8}[state["kind"]](state)


# ------------------------------------------------------------------ work
def work(case):
    kind, t = case["kind"], case["rows"]
    size = 2 if case.get("dtype") == "bf16" else 4
    if kind == "norm":
        h, r = case["width"], case["residual"]
        if case["form"] == "q8":
            # the codes' values come back in 32 bits, one byte of codes and a scale for each row lie below them
            return {"bytes": t * h * (size * (3 if r else 1) + 1) + 4 * t, "flops": 8 * t * h}
        b = t * h * size * (4 if r else 2)
        if case["form"] == "grad":
            b += t * h * size * (3 if r else 2)      # dy (and dz) in, dx out; z is in hand
        return {"bytes": b, "flops": (6 + 10 * (case["form"] == "grad")) * t * h}
    if kind == "route":
        e, k = case["experts"], case["k"]
        return {"bytes": t * e * size * (2 if case["grad"] else 1) + t * k * (12 if case["grad"] else 8),
                "flops": t * e * (8 + 4 * case["grad"])}
    h, f, e, k = case["width"], case["hidden"], case["experts"], case["k"]
    used = min(e, t * k)
    if kind == "experts_q8":
        return {"bytes": used * 3 * f * (h + 1) + t * (3 * h + 4 + 8 * k), "flops": 6.0 * h * f * t * k}
    weights, passes = used * 3 * f * h * size, {"none": 1, "rows": 2, "all": 3}[case["grads"]]
    b = weights * passes + t * h * size * (2 if passes == 1 else 4) + 8 * t * k
    return {"bytes": b, "flops": 6.0 * h * f * t * k * passes}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_norm(s):
    x, w = s["x"].detach().double().requires_grad_(True), s["weight"].detach().double().requires_grad_(True)
    r = s["residual"]
    full = x if r is None else x + r.detach().double()
    # the sum is held in the rows' type: the norm is that of the held values
    held = full + (full.detach().to(s["x"].dtype).double() - full.detach())
    y = held * torch.rsqrt((held * held).mean(1, keepdim=True) + EPS) * w
    if s["form"] == "q8":
        return {"y": None, "z": held.detach()}      # a code next to a half is either neighbour's
    out = {"y": y.detach(), "z": held.detach()}
    if s["form"] == "grad":
        heads, gs = ((y, held), (s["dy"].double(), s["dz"].double())) if r is not None else ((y,), (s["dy"].double(),))
        out["dx"], out["dweight"] = torch.autograd.grad(heads, (x, w), gs)
    return out


def _exact_route(s):
    l = s["logits"].detach().double().requires_grad_(True)
    barred = l.detach() == -math.inf
    if s["score"] == "softmax":
        score = torch.nan_to_num(torch.softmax(l.masked_fill(barred.all(1, keepdim=True), 0.0), 1))
    else:
        score = torch.sigmoid(l)
    c = score.detach() if s["bias"] is None else score.detach() + s["bias"].double()
    c = c.float().double().masked_fill(barred, -math.inf)      # scores that 32 bits do not tell apart are a tie
    t, e = c.shape
    n, per = s["groups"], e // s["groups"]
    best = c.view(t, n, per).topk(s["best"], dim=2)[0]
    rank = best.masked_fill(best == -math.inf, 0.0).sum(2).masked_fill((best == -math.inf).all(2), -math.inf)
    above = (rank.unsqueeze(1) > rank.unsqueeze(2)).sum(2)
    lower = torch.tril(torch.ones(n, n, dtype=torch.bool, device=c.device), -1)
    above = above + ((rank.unsqueeze(1) == rank.unsqueeze(2)) & lower).sum(2)
    c = c.view(t, n, per).masked_fill((above >= s["kept"]).unsqueeze(2) & (n > 1), -math.inf).view(t, e)
    value, index = torch.sort(c, dim=1, descending=True, stable=True)
    value, index = value[:, : s["k"]], index[:, : s["k"]]
    weight = score.gather(1, index).masked_fill(value == -math.inf, 0.0)
    if s["renormalise"]:
        total = weight.sum(1, keepdim=True)
        weight = weight / total.masked_fill(total == 0, 1.0)
    out = {"index": None, "weight": weight.detach()}
    if s["grad"]:
        dl, = torch.autograd.grad(weight, l, s["dweight"].double())
        out["dlogits"] = torch.nan_to_num(dl)
    return out


def _exact_experts(s):
    names = ("x", "weight", "w_in", "w_out")
    x, weight, w_in, w_out = (s[n].detach().double() for n in names)
    f, index = s["hidden"], s["index"]
    y, dx, dweight = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(weight)
    dw_in, dw_out = torch.zeros_like(w_in), torch.zeros_like(w_out)
    dy = s["dy"].double() if s["grads"] != "none" else None
    for e in range(s["experts"]):
        row, slot = torch.nonzero(index == e, as_tuple=True)
        if row.numel() == 0:
            continue
        part = [v.requires_grad_(dy is not None) for v in (x[row], weight[row, slot], w_in[e].clone(), w_out[e].clone())]
        a = part[0] @ part[2].T
        o = (torch.nn.functional.silu(a[:, :f]) * a[:, f:]) @ part[3].T * part[1].unsqueeze(1)
        y.index_add_(0, row, o.detach())
        if dy is not None:
            g = torch.autograd.grad(o, part, dy[row])
            dx.index_add_(0, row, g[0])
            dweight[row, slot] = g[1]
            dw_in[e], dw_out[e] = g[2], g[3]
    out = {"y": y}
    if s["grads"] != "none":
        out["dx"] = dx
    if s["grads"] == "all":
        out |= {"dweight": dweight, "dw_in": dw_in, "dw_out": dw_out}
    return out


def _exact_experts_q8(s):
    f = s["hidden"]
    x = s["x"].double() * s["x_scale"].double()[:, None]
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in range(s["experts"]):
        row, slot = torch.nonzero(s["index"] == e, as_tuple=True)
        if row.numel() == 0:
            continue
        a = x[row] @ (s["w_in"][e].double() * s["w_in_scale"][e].double()[:, None]).T
        h = torch.nn.functional.silu(a[:, :f]) * a[:, f:]
        parts = []
        for lo in range(0, f, GROUP):
            p = h[:, lo:lo + GROUP]
            unit = p.abs().amax(1, keepdim=True).clamp_min(1e-300) / 127
            parts.append(torch.round(p / unit) * unit)
        o = torch.cat(parts, 1) @ (s["w_out"][e].double() * s["w_out_scale"][e].double()[:, None]).T
        y.index_add_(0, row, o * s["weight"][row, slot].double().unsqueeze(1))
    return {"y": y}


def exact(case, seed):
    return {"norm": _exact_norm, "route": _exact_route, "experts": _exact_experts,
            "experts_q8": _exact_experts_q8}[case["kind"]](prepare(case, seed))
