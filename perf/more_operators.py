"""Operators of a training step: what a program hands to them, their plain forms, and the same in 64 bits.

Three operators: the layer norm of per-atom rows (with SiLU, its backward pass and the backward of that, which a loss
on forces needs), the lookup of table rows by species, species pair or token with the gradient summed by token, and
the AdamW step over a model's tensors (states in 32 or 8 bits, gradients clipped by their norm).

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes what a
program holds before the call, ``run(state)`` is one pass, ``work(case)`` what the pass cannot do without and
``exact(case, seed)`` the outputs in 64 bits.  ``own`` selects between the plain form and the framework's calls.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
BLOCK = 256            # values that share a scale in the 8-bit states
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
HYPER = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}


def listed():
    return [
        # ---- layer norm
        # a hidden layer of the energy head, force training on one 32-atom molecule: latency
        {"name": "norm_32x128", "kind": "norm", "rows": 32, "width": 128, "dtype": "fp32", "silu": True, "form": "force"},
        # the head's input norm on the wide (1600) invariants of 10,000 atoms, force training
        {"name": "norm_10000x1600", "kind": "norm", "rows": 10000, "width": 1600, "dtype": "fp32", "silu": False,
         "form": "force"},
        # rows in bfloat16, training on the energies of a large batch
        {"name": "norm_100000x640", "kind": "norm", "rows": 100000, "width": 640, "dtype": "bf16", "silu": False,
         "form": "grad"},
        # widths no vector divides
        {"name": "norm_10007x331", "kind": "norm", "rows": 10007, "width": 331, "dtype": "fp32", "silu": True,
         "form": "force"},
        # ---- lookup
        # a 32-atom molecule's atoms in a table by atomic number: latency
        {"name": "lookup_32x16", "kind": "lookup", "rows": 32, "width": 16, "table": 100, "order": "free",
         "dtype": "fp32", "index": "int64", "scale": 1.0},
        # the first convolution's bias by species pair, 10,000 atoms with 52 neighbours, 64 channels of three ranks
        {"name": "lookup_520000x192", "kind": "lookup", "rows": 520000, "width": 192, "table": 9, "order": "receivers",
         "dtype": "fp32", "index": "int32", "scale": 1.0},
        # the first convolution's weights by species pair, one row for each tile of 16 edges, 2,500 atoms
        {"name": "lookup_8125x12288", "kind": "lookup", "rows": 8125, "width": 12288, "table": 16, "order": "sorted",
         "dtype": "fp32", "index": "int32", "scale": 1.0},
        # a large vocabulary with a long tail and padding, scaled rows of a width no vector divides
        {"name": "lookup_65536x331", "kind": "lookup", "rows": 65536, "width": 331, "table": 30011, "order": "tail",
         "dtype": "bf16", "index": "int64", "scale": math.sqrt(331.0)},
        # ---- optimiser
        # a small sparse trunk (32 channels, two layers)
        {"name": "adamw_trunk_32", "kind": "adamw", "model": "trunk", "channels": 32, "layers": 2, "dtype": "fp32",
         "bits": 32, "max_norm": 0.0},
        # a wide sparse trunk (128 channels, three layers), gradients clipped
        {"name": "adamw_trunk_128", "kind": "adamw", "model": "trunk", "channels": 128, "layers": 3, "dtype": "fp32",
         "bits": 32, "max_norm": 1.0},
        # 16 experts in bfloat16 with 32-bit copies of their weights
        {"name": "adamw_experts_16", "kind": "adamw", "model": "experts", "experts": 16, "width": 640, "hidden": 1280,
         "dtype": "bf16", "bits": 32, "max_norm": 1.0},
        # 32 experts, states in 8 bits
        {"name": "adamw_8bit_experts_32", "kind": "adamw", "model": "experts", "experts": 32, "width": 640,
         "hidden": 1280, "dtype": "fp32", "bits": 8, "max_norm": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "lookup", "adamw"])
    if kind == "norm":
        width = _log(rng, 16, 2048)
        form = rng.choice(["forward", "grad", "force"])
        # the trunks are trained on forces in float32
        return {"kind": kind, "rows": _log(rng, 1, min(100000, 16000000 // width)), "width": width,
                "dtype": "fp32" if form == "force" else rng.choice(["fp32", "bf16"]), "silu": rng.random() < 0.5,
                "form": form}
    if kind == "lookup":
        width = _log(rng, 4, 12288)
        order = rng.choice(["free", "receivers", "sorted", "tail"])
        return {"kind": kind, "rows": _log(rng, 1, min(520000, 90000000 // width)), "width": width,
                "table": _log(rng, 2, min(50000 if order in ("free", "tail") else 256, 20000000 // width)), "order": order,
                "dtype": rng.choice(["fp32", "bf16"]), "index": rng.choice(["int32", "int64"]),
                "scale": rng.choice([1.0, math.sqrt(width)])}
    c = {"kind": kind, "dtype": rng.choice(["fp32", "bf16"]), "bits": rng.choice([32, 8]),
         "max_norm": rng.choice([0.0, 1.0, 1000.0])}
    if rng.random() < 0.5:
        channels = rng.choice([32, 64, 128])
        return c | {"model": "trunk", "channels": channels, "layers": rng.randint(2, 3 if channels == 128 else 4)}
    width, hidden = _log(rng, 32, 1600), _log(rng, 32, 1280)
    return c | {"model": "experts", "experts": _log(rng, 2, max(2, min(64, 60000000 // (3 * width * hidden)))),
                "width": width, "hidden": hidden}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _sizes(case):
    """Values in each tensor of the model: a sparse trunk's parameters, or an expert layer's."""
    if case["model"] == "experts":
        e, h, f = case["experts"], case["width"], case["hidden"]
        return [h, 100 * e, e * 2 * f * h, e * h * f]
    c, n = case["channels"], case["layers"]
    out = [160, 1024, 64, 512, 8]
    for layer in range(n):
        w = 6 * c * (64 if layer == 0 else c)
        out += [512, 64, 4096, 64, 64 * w, w]
    s, wide = 32 * (n - 1), c * n
    out += [s * wide * wide] * 3
    k = 3 * wide + s
    out += [k, k]
    for _ in range(3):
        out += [128 * k, 128, 128, 128]
        k = 128
    return out + [17 * 128, 17, 17]


def _index(g, case):
    t, v, order = case["rows"], case["table"], case["order"]
    if order in ("receivers", "sorted"):
        s = max(1, math.isqrt(v))
        kind = torch.randint(0, s, (t // 52 + 1,), generator=g, device=DEV).repeat_interleave(52)[:t]
        at = (torch.randint(0, s, (t,), generator=g, device=DEV) * s + kind).clamp(max=v - 1)
        at = torch.sort(at)[0] if order == "sorted" else at
    elif order == "tail":
        u = torch.rand(t, generator=g, device=DEV)
        at = (torch.exp(u * math.log(v + 1.0)) - 1).long().clamp(max=v - 1)
        at = torch.randperm(v, generator=g, device=DEV)[at]
        at = torch.where(torch.rand(t, generator=g, device=DEV) < 1 / 16, -1, at)     # padding
    else:
        at = torch.randint(0, v, (t,), generator=g, device=DEV)
    return at.to(torch.int32 if case["index"] == "int32" else torch.int64)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["kind"] == "norm":
        t, h, dt = case["rows"], case["width"], DTYPES[case["dtype"]]
        # rows of different sizes and means, as the invariants of different species are
        size = torch.exp(0.5 * _randn(g, t, 1))
        s["x"] = (size * (_randn(g, t, h) + _randn(g, t, 1))).to(dt).requires_grad_(True)
        s["weight"] = (1 + 0.2 * _randn(g, h)).to(dt).requires_grad_(True)
        s["bias"] = (0.1 * _randn(g, h)).to(dt).requires_grad_(True)
        if case["form"] != "forward":
            s["dy"] = _randn(g, t, h).to(dt)
        if case["form"] == "force":
            s["dy"].requires_grad_(True)
            s["ey"], s["ex"] = _randn(g, t, h).to(dt), _randn(g, t, h).to(dt)
        return s
    if case["kind"] == "lookup":
        t, d, v, dt = case["rows"], case["width"], case["table"], DTYPES[case["dtype"]]
        s["index_of"] = _index(g, case)
        s["weight"] = _randn(g, v, d).to(dt).requires_grad_(True)
        s["dy"] = _randn(g, t, d).to(dt)
        return s
    # every tensor of the model lies in one buffer, each at a multiple of 256 values
    sizes = _sizes(case)
    room = [-(-n // BLOCK) * BLOCK for n in sizes]
    starts = [sum(room[:i]) for i in range(len(room))]
    total, dt = sum(room), DTYPES[case["dtype"]]
    tensor = torch.arange(len(room), device=DEV).repeat_interleave(torch.tensor(room, device=DEV), output_size=total)
    first = torch.tensor(starts, device=DEV)
    place = torch.arange(total, device=DEV) - first[tensor]
    there = place < torch.tensor(sizes, device=DEV)[tensor]
    # gradients and states of tensors of different sizes
    size = torch.exp(2.0 * _randn(g, len(sizes)) - 7)[tensor] * there
    full = 0.05 * _randn(g, total) * there
    s["flat"] = {"p": full.to(dt), "g": (size * _randn(g, total)).to(dt)}
    if case["dtype"] == "bf16":
        s["flat"]["master"] = full
    m, r = 0.3 * size * _randn(g, total), size * (0.2 + torch.rand(total, generator=g, device=DEV))
    if case["bits"] == 32:
        s["flat"] |= {"m": m, "v": r * r}
    else:
        half = torch.full_like(place, 1 << 31)
        s["flat"]["m_code"], s["flat"]["m_scale"] = _encode(m, half, True)
        s["flat"]["r_code"], s["flat"]["r_scale"] = _encode(r, half, False)
    s["step"] = torch.full((len(sizes),), 1000.0 + seed % 1000, device=DEV)
    s["steps"] = list(s["step"].unbind())
    for name, flat in s["flat"].items():
        per = BLOCK if name.endswith("_scale") else 1
        s[name] = [flat[a // per:a // per + -(-n // per)] for a, n in zip(starts, sizes)]
    s["place"] = place
    return s


# ------------------------------------------------------------------ plain forms
def _plain_norm(s):
    dt, force = s["x"].dtype, s["form"] == "force"
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()

    def mean(v):
        return v.mean(-1, keepdim=True)

    mu = mean(x.double()).float()
    c = x - mu
    r = 1 / torch.sqrt(mean(c * c) + EPS)
    zh = c * r
    u = zh * w + b
    if s["silu"]:
        sig = 1 / (1 + torch.exp(-u))
        y, d1, d2 = u * sig, sig * (1 + u * (1 - sig)), sig * (1 - sig) * (2 + u * (1 - 2 * sig))
    else:
        y, d1, d2 = u, torch.ones_like(u), torch.zeros_like(u)
    out = {"y": y.to(dt)}
    if s["form"] == "forward":
        return out

    def back(dy):
        """(dx, dweight, dbias) without rounding."""
        du = dy * d1
        gg = du * w
        return r * (gg - mean(gg) - zh * mean(gg * zh)), (du * zh).sum(0), du.sum(0)

    dy = s["dy"].float()
    dx, dw, db = back(dy)
    out["dx"] = dx.to(dt)
    if not force:
        return out | {"dweight": dw.to(dt), "dbias": db.to(dt)}
    # loss = ex . dx(x, dy, weight, bias) + ey . y
    v = s["ex"].float()
    du = dy * d1
    gg = du * w
    q = r * (v - mean(v) - zh * mean(v * zh))
    a = w * q
    e = dy * d2 * a
    k = e * w - r * (gg * mean(v * zh) + v * mean(gg * zh))
    turn = mean(gg * v) - mean(gg) * mean(v) - mean(gg * zh) * mean(v * zh)
    gx = r * (k - mean(k) - zh * mean(k * zh)) - r * r * zh * turn
    ex, ew, eb = back(s["ey"].float())
    return out | {"grad_x": (gx + ex).to(dt), "grad_weight": ((du * q + e * zh).sum(0) + ew).to(dt),
                  "grad_bias": (e.sum(0) + eb).to(dt), "grad_dy": (d1 * a).to(dt)}


def _plain_lookup(s):
    dt, v = s["weight"].dtype, s["table"]
    index = s["index_of"].long()
    there = ((index >= 0) & (index < v)).unsqueeze(1)
    at = torch.where(there.squeeze(1), index, 0)
    table = s["scale"] * s["weight"].float()
    y = torch.where(there, table[at], 0.0)
    dy = s["dy"].float()
    if v <= 256:
        chosen = (index.unsqueeze(0) == torch.arange(v, device=index.device).unsqueeze(1)).float()
        total = s["scale"] * (chosen @ dy)
    else:
        total = torch.zeros(v, dy.shape[1], dtype=torch.float64, device=dy.device)
        total.index_add_(0, at, torch.where(there, dy, 0.0).double())
        total = s["scale"] * total
    return {"y": y.to(dt), "dtable": total.to(dt)}


def _hash(place, step):
    """32 bits from a value's number in its tensor and the step."""
    low = 0xFFFFFFFF
    h = (place * 0x9E3779B1 + step * 0x6A09E667) & low
    h = h ^ (h >> 16)
    h = (h * 0xBB67AE85) & low
    h = h ^ (h >> 15)
    h = (h * 0x3C6EF373) & low
    return h ^ (h >> 16)


def _encode(value, bits, signed):
    """8-bit floats with a scale for each 256 values, the largest of them: a sign, 4 exponent and 3 fraction bits, or
    4 and 4 without a sign; the random ``bits`` added below the last one kept make the rounding's mean the value.  A
    value above zero without a sign has a code above zero; values whose largest is below 2^-100 are zeros."""
    shift, most = (20, 127) if signed else (19, 255)
    base = (0x3F800000 >> shift) - most
    size = value.abs().view(-1, BLOCK)
    top = size.amax(1, keepdim=True)
    top = torch.where(top >= 2.0 ** -100, top, 0.0)
    over = torch.where(top > 0, 1 / top.double(), 0.0).float()
    y = (size * over).clamp(max=1.0).view(-1)
    add = (bits & 0xFFFFF) if signed else bits >> 13
    code = (((y.view(torch.int32).long() + add) >> shift) - base).clamp(0, most)
    if not signed:
        code = torch.where(y > 0, code.clamp(min=1), 0)
    else:
        code = code + 128 * (value < 0).long()
    return code.to(torch.uint8), top.squeeze(1)


def _decode(code, scale, signed):
    shift, most = (20, 127) if signed else (19, 255)
    base = (0x3F800000 >> shift) - most
    size = code.to(torch.int32) & most
    y = torch.where(size > 0, ((size + base) << shift).view(torch.float32), 0.0)
    if signed:
        y = torch.where(code >= 128, -y, y)
    return (y.view(-1, BLOCK) * scale.unsqueeze(1)).view(-1)


def _plain_adamw(s):
    f, n = s["flat"], s["place"].numel()
    b1, b2 = HYPER["betas"]
    lr = HYPER["lr"]
    g = f["g"].float()
    out = {}
    if s["max_norm"]:
        norm = torch.sqrt(g.double().square().sum()).float()
        out["norm"] = norm
        g = g * (s["max_norm"] / (norm.double() + 1e-6)).clamp(max=1.0).float()
    s["step"].add_(1)
    # one step count for each tensor, all the same here
    t = s["step"][:1].double()
    size, over = (lr / (1 - b1 ** t)).float(), (1 / torch.sqrt(1 - b2 ** t)).float()
    if s["bits"] == 32:
        m, v = f["m"], f["v"]
    else:
        m, root = _decode(f["m_code"], f["m_scale"], True), _decode(f["r_code"], f["r_scale"], False)
        v = root * root
    m = b1 * m + (1 - b1) * g
    v = b2 * v + ((1 - b2) * g) * g
    root = torch.sqrt(v.double()).float()
    p = f["p"] if "master" not in f else f["master"]
    p = p * (1 - lr * HYPER["weight_decay"]) - size * (m / (root * over + HYPER["eps"]))
    f["p"].copy_(p)
    out["p"] = f["p"]
    if "master" in f:
        f["master"].copy_(p)
        out["master"] = f["master"]
    if s["bits"] == 32:
        f["m"].copy_(m)
        f["v"].copy_(v)
        return out | {"m": f["m"], "v": f["v"]}
    bits = _hash(s["place"], t.long())
    for name, value, signed in (("m", m, True), ("r", root, False)):
        code, scale = _encode(value, bits, signed)
        f[name + "_code"].copy_(code)
        f[name + "_scale"].copy_(scale)
        out[name] = _decode(f[name + "_code"], f[name + "_scale"], signed)
    return out


# ------------------------------------------------------------------ the framework's calls
def _own_norm(s):
    from fsctep_amd import learn_ops as L
    x, w, b = s["x"], s["weight"], s["bias"]
    act = "silu" if s["silu"] else None
    if s["form"] == "forward":
        with torch.no_grad():
            return {"y": L.layer_norm(x, w, b, EPS, act)}
    y = L.layer_norm(x, w, b, EPS, act)
    if s["form"] == "grad":
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    dx, = torch.autograd.grad(y, x, s["dy"], create_graph=True)
    gx, gw, gb, gdy = torch.autograd.grad((dx, y), (x, w, b, s["dy"]), (s["ex"], s["ey"]))
    return {"y": y, "dx": dx, "grad_x": gx, "grad_weight": gw, "grad_bias": gb, "grad_dy": gdy}


def _own_lookup(s):
    from fsctep_amd import learn_ops as L
    y = L.embedding(s["weight"], s["index_of"], s["scale"])
    return {"y": y, "dtable": torch.autograd.grad(y, s["weight"], s["dy"])[0]}


def _own_adamw(s):
    from fsctep_amd import optim
    f = s["flat"]
    more = {"max_norm": s["max_norm"] or None, "masters": s.get("master"), **HYPER}
    if s["bits"] == 32:
        norm = optim.adamw_step(s["p"], s["g"], s["m"], s["v"], s["steps"], **more)
        out = {"m": f["m"], "v": f["v"]}
    else:
        norm = optim.adamw_step_q8(s["p"], s["g"], s["m_code"], s["m_scale"], s["r_code"], s["r_scale"], s["steps"],
                                   **more)
        out = {"m": optim.moment_values(f["m_code"], f["m_scale"]), "r": optim.root_values(f["r_code"], f["r_scale"])}
    out["p"] = f["p"]
    if s["max_norm"]:
        out["norm"] = norm
    if "master" in f:
        out["master"] = f["master"]
    return out


def run(state):
    if own:
        return {"norm": _own_norm, "lookup": _own_lookup, "adamw": _own_adamw}[state["kind"]](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "lookup": _plain_lookup, "adamw": _plain_adamw}[state["kind"]](state)


# ------------------------------------------------------------------ work
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": n * size * {"forward": 2, "grad": 4, "force": 8}[case["form"]],
                "flops": n * {"forward": 8, "grad": 22, "force": 70}[case["form"]]}
    if case["kind"] == "lookup":
        t, d, v = case["rows"], case["width"], case["table"]
        return {"bytes": size * d * (2 * t + min(v, t) + v) + t * (4 if case["index"] == "int32" else 8), "flops": 2 * t * d}
    n = sum(_sizes(case))
    # parameter (in bfloat16 its copy, too) and states in and out, the gradient in: 28 bytes a value in either type, 16
    # with states in 8 bits; what those stand for comes back in 32 bits
    return {"bytes": n * (28 if case["bits"] == 32 else 24), "flops": 16 * n}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_norm(s):
    x, w, b = (s[n].detach().double().requires_grad_(True) for n in ("x", "weight", "bias"))
    h = x.shape[1]
    u = torch.nn.functional.layer_norm(x, (h,), w, b, EPS)
    y = torch.nn.functional.silu(u) if s["silu"] else u
    out = {"y": y.detach()}
    if s["form"] == "forward":
        return out
    dy = s["dy"].detach().double().requires_grad_(True)
    if s["form"] == "grad":
        out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(y, (x, w, b), dy)
        return out
    dx, = torch.autograd.grad(y, x, dy, create_graph=True)
    out["dx"] = dx.detach()
    # the held dx has no rounding of its own here
    got = torch.autograd.grad((dx, y), (x, w, b, dy), (s["ex"].double(), s["ey"].double()))
    out["grad_x"], out["grad_weight"], out["grad_bias"], out["grad_dy"] = got
    return out


def _exact_lookup(s):
    w = s["weight"].detach().double()
    padded = torch.cat([w, w.new_zeros(1, w.shape[1])])
    index = s["index_of"].long()
    index = torch.where((index < 0) | (index >= s["table"]), s["table"], index)
    y = s["scale"] * padded[index]
    order = torch.argsort(index)
    counts = torch.bincount(index, minlength=s["table"] + 1).tolist()
    dtable = torch.zeros_like(padded)
    if s["table"] <= 4096:
        at = 0
        for k, n in enumerate(counts):
            if n:
                dtable[k] = s["dy"][order[at:at + n]].double().sum(0)
            at += n
    else:
        dtable.index_put_((index,), s["dy"].double(), accumulate=True)
    return {"y": y, "dtable": s["scale"] * dtable[:-1]}


def _exact_adamw(s):
    f = {k: v.double() if v.is_floating_point() else v for k, v in s["flat"].items()}
    (b1, b2), lr, eps, wd = HYPER["betas"], HYPER["lr"], HYPER["eps"], HYPER["weight_decay"]
    g, out = f["g"], {}
    if s["max_norm"]:
        norm = float(torch.linalg.vector_norm(g))
        out["norm"] = torch.tensor(norm, dtype=torch.float64, device=g.device)
        g = g * min(1.0, s["max_norm"] / (norm + 1e-6))
    t = float(s["step"][0]) + 1
    if s["bits"] == 32:
        m, v = f["m"], f["v"]
    else:
        def value(code, scale, fraction):
            """(1 + c / 2^fraction) 2^e of a code, with the largest code at 1."""
            size = code.long() & (127 if fraction == 3 else 255)
            steps = size - (127 if fraction == 3 else 255)
            e = torch.div(steps, 1 << fraction, rounding_mode="floor")
            y = (1 + (steps - (e << fraction)).double() / (1 << fraction)) * torch.exp2(e.double())
            y = torch.where(size > 0, y, 0.0) * scale.repeat_interleave(BLOCK)
            return torch.where((code >= 128) & (fraction == 3), -y, y)
        m = value(f["m_code"], f["m_scale"], 3)
        v = value(f["r_code"], f["r_scale"], 4) ** 2
    m = m + (1 - b1) * (g - m)
    v = v + (1 - b2) * (g * g - v)
    p = f["master"] if "master" in f else f["p"]
    p = p - lr * wd * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    out["p"] = p
    if "master" in f:
        out["master"] = p
    # an 8-bit state next to a border is either neighbour's
    return out | ({"m": m, "v": v} if s["bits"] == 32 else {"m": None, "r": None})


def exact(case, seed):
    return {"norm": _exact_norm, "lookup": _exact_lookup, "adamw": _exact_adamw}[case["kind"]](prepare(case, seed))
