"""The training step's operators through the C ABI, every output and workspace of the size that is asked for inside a larger
buffer whose bytes around it have to stay, at odd addresses too; results as the torch ops give them."""

import ctypes
import math

import pytest
import torch

from fsctep_amd import _lib, learn_ops as L, optim
from test_learn_gpu import BF16, DEV, EPS, F32, LOOKUPS, gen, norm_inputs, randn, tokens
from test_learn_host import Adam, Settings

pytestmark = pytest.mark.gpu
GUARD = 1 << 16
FILL = 0xA5


class Guarded:
    """``shape`` values of a type between guard bytes, ``off`` values behind a 16-byte boundary; holding ``like`` or 0xA5."""

    def __init__(self, shape, dtype, off=0, like=None):
        size = torch.empty(0, dtype=dtype).element_size()
        self.a = GUARD + off * size
        self.n = size * math.prod(shape)
        self.buf = torch.full((2 * GUARD + self.n + 64,), FILL, dtype=torch.uint8, device=DEV)
        if self.n:
            raw = self.buf[self.a:self.a + self.n]
            self.t = (raw.view(dtype) if self.a % size == 0 else raw).view(shape)
            if like is not None:
                self.t.copy_(like)
        else:
            self.t = torch.empty(shape, dtype=dtype, device=DEV)
        self.ptr = self.buf.data_ptr() + self.a

    def check(self, what):
        assert int((self.buf[:self.a] != FILL).sum()) == 0, f"{what}: bytes before"
        assert int((self.buf[self.a + self.n:] != FILL).sum()) == 0, f"{what}: bytes behind"


def stream():
    return _lib.stream_handle(torch.device(DEV))


def code(dtype):
    return 0 if dtype == F32 else 1


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 3), (2, 7), (5, 9), (17, 64), (33, 65), (4, 128), (130, 331), (70, 384), (9, 640),
                                        (21, 770), (5, 1024), (3, 1600), (2, 2049), (1025, 96), (0, 50), (3, 4097), (2, 5003), (1026, 4100),
                                        (2, 8192), (1, 8193)])
def test_layer_norm_writes_its_outputs_alone(rows, width, dtype, off):
    a = norm_inputs(max(rows, 1), width, dtype, dtype)
    a = {k: (t[:rows] if t.dim() == 2 else t) for k, t in a.items()}
    ins = {k: Guarded(t.shape, dtype, off, t) for k, t in a.items()}
    n = ctypes.c_int64()
    _lib.call("fsc_layer_norm_workspace", rows, width, ctypes.byref(n))
    out = {k: Guarded((rows, width), dtype, off) for k in ("y", "dx", "gx", "gdy")}
    out |= {k: Guarded((width,), dtype, off) for k in ("dw", "db", "gw", "gb")}
    out |= {"mean": Guarded((rows,), torch.float64), "rstd": Guarded((rows,), F32), "ws": Guarded((n.value,), F32)}
    p = lambda k: (ins.get(k) or out.get(k)).ptr  # noqa: E731
    c = code(dtype)
    _lib.call("fsc_layer_norm_forward", rows, width, c, c, 1, width, p("x"), p("w"), p("b"), EPS, p("y"), p("mean"), p("rstd"), stream())
    _lib.call("fsc_layer_norm_backward", rows, width, c, c, 1, width, width, width, p("x"), p("w"), p("b"), EPS, p("mean"), p("rstd"),
              p("dy"), p("v"), p("dx"), p("dw"), p("db"), p("ws"), stream())
    _lib.call("fsc_layer_norm_backward_twice", rows, width, c, c, 1, width, width, width, p("x"), p("w"), p("b"), EPS, p("mean"),
              p("rstd"), p("dy"), p("v"), p("vw"), p("vb"), p("gx"), p("gdy"), p("gw"), p("gb"), p("ws"), stream())
    torch.cuda.synchronize()
    for k, g in (ins | out).items():
        g.check(k)
    for k, t in a.items():
        assert torch.equal(ins[k].t, t), k
    x, w, b = a["x"], a["w"], a["b"]
    y, mean, rstd = torch.ops.fsctep.layer_norm(x, w, b, EPS, 1, True)
    first = torch.ops.fsctep.layer_norm_backward(a["dy"], x, w, b, mean, rstd, EPS, 1, True, True, True, a["v"])
    second = torch.ops.fsctep.layer_norm_backward_twice(a["v"], a["vw"], a["vb"], a["dy"], x, w, b, mean, rstd, EPS, 1, True, True,
                                                        True, True)
    for k, t in zip(("y", "dx", "dw", "db", "gx", "gdy", "gw", "gb"), (y, *first, *second)):
        assert torch.equal(out[k].t, t), k


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["free", "outside", "one"])
@pytest.mark.parametrize("rows,width,table", LOOKUPS + [(2000, 1, 3), (1500, 2, 40), (3000, 257, 20), (3000, 259, 700), (5000, 5, 33)])
def test_lookup_writes_its_outputs_alone(rows, width, table, kind, dtype, off):
    g = gen(rows + width)
    index = tokens(g, rows, table, torch.int64, kind)
    t, dy = Guarded((table, width), dtype, off, randn(g, table, width, dtype=dtype)), Guarded((rows, width), dtype, off, randn(g, rows, width, dtype=dtype))
    n = ctypes.c_int64()
    _lib.call("fsc_embedding_workspace", rows, width, table, ctypes.byref(n))
    y, dt, ws = Guarded((rows, width), dtype, off), Guarded((table, width), dtype, off), Guarded((n.value,), torch.uint8)
    i = Guarded((rows,), torch.int64, 0, index)
    _lib.call("fsc_embedding_forward", rows, width, table, code(dtype), 64, width, t.ptr, i.ptr, 1.5, y.ptr, stream())
    _lib.call("fsc_embedding_backward", rows, width, table, code(dtype), 64, width, dy.ptr, i.ptr, 1.5, dt.ptr, ws.ptr, stream())
    torch.cuda.synchronize()
    for name, b in dict(table=t, dy=dy, y=y, dtable=dt, ws=ws, index=i).items():
        b.check(name)
    assert torch.equal(y.t, L.embedding(t.t.clone(), index, 1.5))
    assert torch.equal(dt.t, torch.ops.fsctep.embedding_backward(dy.t.clone(), index, table, 1.5))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_step_writes_its_tensors_alone(bits, dtype, off):
    g = gen(3)
    sizes = [1, 2, 3, 4, 5, 255, 256, 257, 1023, 2047, 2048, 2049, 8191, 8192, 8193, 0, 5000] * 4        # more than one launch takes
    state = F32 if bits == 32 else torch.uint8
    hold, entries, twins = [], [], []
    for n in sizes:
        groups = -(-n // 256)
        v = dict(p=randn(g, n).to(dtype), g=randn(g, n).to(dtype), m=torch.zeros(n, dtype=state, device=DEV),
                 v=torch.zeros(n, dtype=state, device=DEV), m_scale=torch.zeros(groups, device=DEV), v_scale=torch.zeros(groups, device=DEV),
                 master=randn(g, n), step=torch.zeros((), device=DEV))
        b = {k: Guarded(t.shape, t.dtype, off if k not in ("m_scale", "v_scale", "step") else 0, t) for k, t in v.items()}
        hold.append(b)
        twins.append({k: t.clone() for k, t in v.items()})
        entries.append(Adam(n, code(dtype), 0, *(b[k].ptr for k in ("p", "g", "m", "v", "m_scale", "v_scale", "master", "step"))))
    array = (Adam * len(sizes))(*entries)
    a, c = ctypes.c_int64(), ctypes.c_int64()
    _lib.call("fsc_adamw_workspace", len(sizes), array, ctypes.byref(a), ctypes.byref(c))
    step_ws, norm_ws, norm = Guarded((a.value,), torch.uint8), Guarded((c.value,), torch.uint8), Guarded((1,), F32)
    rule = Settings(1e-2, 0.9, 0.99, 1e-8, 0.1, 0.5, None, norm.ptr, bits, 0)
    for _ in range(2):
        _lib.call("fsc_grad_norm", len(sizes), array, norm_ws.ptr, norm.ptr, stream())
        _lib.call("fsc_adamw_step", len(sizes), array, ctypes.byref(rule), step_ws.ptr, stream())
    torch.cuda.synchronize()
    for b in (step_ws, norm_ws, norm):
        b.check("workspace")
    for i, b in enumerate(hold):
        for k, t in b.items():
            t.check(f"{k} of {sizes[i]}")
    pick = lambda k: [t[k] for t in twins]  # noqa: E731
    more = dict(lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1, max_norm=0.5, masters=pick("master") if dtype == BF16 else None)
    for _ in range(2):
        if bits == 32:
            got = optim.adamw_step(pick("p"), pick("g"), pick("m"), pick("v"), pick("step"), **more)
        else:
            got = optim.adamw_step_q8(pick("p"), pick("g"), pick("m"), pick("m_scale"), pick("v"), pick("v_scale"), pick("step"), **more)
    assert torch.equal(norm.t[0], got)
    for i, (b, t) in enumerate(zip(hold, twins)):
        for k in t:
            assert torch.equal(b[k].t.view(t[k].shape), t[k]), (k, sizes[i])


@pytest.mark.parametrize("root", [0, 1])
@pytest.mark.parametrize("n", [1, 255, 256, 4096, 4097, 10001])
def test_values_write_their_output_alone(n, root):
    g = gen(n)
    c = Guarded((n,), torch.uint8, 3, torch.randint(0, 256, (n,), generator=g, device=DEV).to(torch.uint8))
    s, v = Guarded((-(-n // 256),), F32, 0, torch.rand(-(-n // 256), generator=g, device=DEV)), Guarded((n,), F32, 1)
    _lib.call("fsc_adamw_values", n, root, c.ptr, s.ptr, v.ptr, stream())
    torch.cuda.synchronize()
    for b in (c, s, v):
        b.check("values")
    assert torch.equal(v.t, torch.ops.fsctep.adamw_values(c.t.clone(), s.t.clone(), bool(root)))
