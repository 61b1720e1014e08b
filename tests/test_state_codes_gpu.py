"""The 8-bit states of gradients that span far more than a block's codes, on the GPU: those of the oracle to the bit."""

import numpy as np
import pytest
import torch

from fsctep_amd import optim
from oracle import learn as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("step", [0, 7, 4096])
@pytest.mark.parametrize("low", [-14, -17, -30, -60])
def test_codes_of_blocks_that_span_the_range(low, step):
    """From states of zeros, m and sqrt(v) are the gradient times a number: their codes at and below the first one."""
    n = 2048
    rng = np.random.default_rng(step - low)
    g = np.exp2(rng.uniform(low, 0, n)) * rng.choice([-1.0, 1.0], n)
    g[::256] = 1.0
    # around code 1, and one spacing below it
    g[1::256], g[2::256], g[3::256], g[4::256] = 1.25 * 2.0 ** -16, -1.249 * 2.0 ** -16, 1.126 * 2.0 ** -16, 1.12 * 2.0 ** -16
    g = g.astype(np.float32)
    p, t = torch.zeros(n, device=DEV), torch.full((), float(step), device=DEV)
    codes = [torch.zeros(n, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(n // 256, device=DEV) for _ in range(2)]
    optim.adamw_step_q8([p], [torch.from_numpy(g).to(DEV)], [codes[0]], [scales[0]], [codes[1]], [scales[1]], [t], betas=(0.5, 0.75))
    f = np.float32
    for k, (value, root) in enumerate(((f(0.5) * g, False), (np.sqrt(f(0.25) * g * g), True))):
        code, scale = O.encode(value, step + 1, root)
        assert np.array_equal(scales[k].cpu().numpy(), scale) and np.array_equal(codes[k].cpu().numpy(), code), root
    assert torch.isfinite(p).all()
