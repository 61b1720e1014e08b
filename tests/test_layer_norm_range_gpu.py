"""The layer norm of rows whose squares leave the range of 32 bits, on the GPU against 64 bits."""

import pytest
import torch

from oracle import learn as O
from test_learn_gpu import BF16, EPS, F32, U, close, norm_check, norm_inputs

pytestmark = pytest.mark.gpu
# every shape of a row in registers, its block, and those that are read again
SHAPES = [(40, 20), (7, 64), (33, 100), (9, 150), (17, 300), (20, 331), (9, 500), (9, 640), (5, 700), (5, 1000), (6, 1600), (3, 2048), (4, 4000),
          (3, 8000), (3, 3), (2, 9000)]


@pytest.mark.parametrize("exponent", [40, 60, 62, 64, 80, 120])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", SHAPES)
def test_rows_of_large_values(rows, width, dtype, exponent):
    """Deviations up to 2^124: the norm and its gradients are what they are of ordinary rows, at the tolerance of those."""
    a = norm_inputs(rows, width, dtype, F32)
    # the rows' own sizes spread over a factor of four or so: clipped, so that none leaves the type
    a["x"] = (a["x"].float().clamp(-8, 8) * 2.0 ** exponent).to(dtype)
    norm_check(silu=True, **a)
    a["x"][1:] = a["x"][1:] * 2.0 ** -exponent          # beside ordinary rows, in the same wave
    norm_check(silu=False, **a)


@pytest.mark.parametrize("exponent", [-40, -60, -70, -100])
@pytest.mark.parametrize("rows,width", SHAPES)
def test_rows_of_small_values_without_eps(rows, width, exponent):
    """The root is of the squares alone."""
    a = norm_inputs(rows, width, F32, F32)
    x = a["x"] * 2.0 ** exponent
    y, mean, rstd = torch.ops.fsctep.layer_norm(x, a["w"], a["b"], 0.0, 0, True)
    want = O.layer_norm(x.double(), a["w"].double(), a["b"].double(), 0.0, False)
    size = O.norm_sizes(x, a["w"], a["b"], 0.0, False, a["dy"], a["v"])["y"]
    close(y, want, size, 50 + width / 64, f"y of {rows} x {width}")
    c = x.double() - x.double().mean(1, keepdim=True)
    r = 1 / c.square().mean(1).sqrt()
    assert ((rstd.double() - r).abs() <= (50 + width / 64) * U * r).all()


def test_rows_without_a_deviation():
    """Nothing but the mean: the bias with an eps, however small the squares of nothing are."""
    x = torch.tensor([0.0, 3.0, -2.0 ** 100], device="cuda").unsqueeze(1).expand(3, 640)
    b = torch.linspace(-1, 1, 640, device="cuda")
    for eps in (EPS, 1e-30):
        assert torch.equal(torch.ops.fsctep.layer_norm(x, None, b, eps, 0, False)[0], b.expand(3, 640))
